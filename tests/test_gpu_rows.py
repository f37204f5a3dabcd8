"""Layer normalisation, row quantisation and the 8-bit product (yolo_amd.ops) against plain 64-bit implementations.

Tolerances are bounds on the rounding errors, written out where they are used: u = 2^-24 is half a step of fp32, half(t) half
a step of the stored type relative to the value.  A row's fp32 sum goes through at most 32 values one after the other in a lane and
a tree of 8 levels: its error is at most 40 u times the sum of magnitudes.
"""
import math

import pytest
import torch

from yolo_amd import _ffi, engine, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16


def half(t):
    return torch.finfo(t).eps / 2


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def within(got, want, bound):
    """|got - want| <= bound everywhere; infinities and NaN in the same places."""
    got, want = got.double(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
    over = (got - want).abs()[fine] - bound.expand_as(want)[fine]
    assert over.numel() == 0 or over.max() <= 0, f"off by {over.max():.3g} over the bound at most"


# ---- plain implementations in 64 bits --------------------------------------------------------------------------------------
def norm64(x, w, b, eps):
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
    xh = (x - mean) * rstd
    y = xh
    if w is not None:
        y = y * w.double()
    if b is not None:
        y = y + b.double()
    return y, xh, rstd


def xh_error(x, xh, rstd):
    """Bound on the error of (x - mean) * rstd in fp32: the mean is off by at most 41 u mean|x|, the variance by 44 u of itself
    (a shift of the mean moves it in second order only), rstd by 25 u, two more roundings."""
    return 64 * U * (x.double().abs().mean(-1, keepdim=True) * rstd + xh.abs())


def quant64(v):
    """(q, scale) of rows in 64 bits, from the definition."""
    v = v.double()
    top = v.abs().amax(-1)
    bad = ~torch.isfinite(v).all(-1)
    top = torch.where(bad, 0.0, top.nan_to_num(0.0, 0.0, 0.0))
    some = top >= float(torch.tensor(127.0) * torch.tensor(1.17549435e-38))
    s = torch.where(some, (top / 127).float().double(), 1.0)
    q = torch.round(torch.where(some[..., None], v, 0.0) / s[..., None])
    scale = torch.where(some, s, 0.0)
    scale[bad] = float("nan")
    return q.to(torch.int8), scale.float()


def product64(q, s, wq, ws, bias, act, slope, res, mode):
    """(y, bound without the stored type's half step)."""
    acc = q.double() @ wq.double().t().contiguous()          # exact: integers below 2^53
    p = acc * s.double()[..., None] * ws.double()
    b = bias.double() if bias is not None else torch.zeros_like(ws).double()
    v = p + b
    e = 5 * U * (p.abs() + b.abs())               # the sum's conversion, two products, the sum with the bias
    if res is not None and mode == "before":
        v = v + res.double()
        e = e + U * (v.abs() + p.abs() + b.abs())
    if act == "silu":
        # exp2 and reciprocal of the hardware are one step (2 u) off each, exp2's argument two roundings of |v| log2(e)
        y = v * torch.sigmoid(v)
        e = 1.1 * e + (3 * v.abs() + 8) * U * y.abs()
    elif act == "leaky":
        y = torch.where(v > 0, v, v * float(torch.tensor(slope, dtype=F32)))
        e = e * max(1.0, abs(slope)) + U * y.abs()
    else:
        y = v
    if res is not None and mode == "after":
        e = e + U * (y.abs() + res.double().abs())
        y = y + res.double()
    return y, e


# ---- layer norm ----------------------------------------------------------------------------------------------------------
SIZES = [(1, 1), (1, 16), (3, 7), (5, 8), (64, 24), (257, 32), (1, 75), (33, 64), (129, 128), (17, 255), (400, 512), (65, 513), (9, 1000),
         (31, 1024), (12, 2048), (7, 2050), (3, 4096), (2, 5001), (2, 8192)]


@pytest.mark.parametrize("dtype,pdtype", [(F32, F32), (BF16, F32), (BF16, BF16), (F32, BF16)])
@pytest.mark.parametrize("rows,C", SIZES)
def test_layer_norm_forward_and_backward(rows, C, dtype, pdtype):
    g = gen(rows * 10007 + C)
    x = (randn(g, rows, C) * (0.2 + randn(g, C).abs()) + randn(g, C)).to(dtype)
    w, b = (1 + 0.3 * randn(g, C)).to(pdtype), (0.3 * randn(g, C)).to(pdtype)
    dy = randn(g, rows, C, dtype=dtype)
    eps = 1e-5
    y64, xh, rstd = norm64(x, w, b, eps)
    ex = xh_error(x, xh, rstd)
    y, mean, rs = ops.layer_norm_forward(x, w, b, eps)
    assert y.dtype == dtype and mean.shape == rs.shape == (rows,)
    # y = xh w + b: one fused rounding on top of xh's error, then the stored type's
    within(y, y64, ex * w.double().abs() + 2 * U * ((xh * w.double()).abs() + b.double().abs()) + half(dtype) * y64.abs() * (1 + 1e-6) + 1e-30)
    assert torch.equal(y, ops.layer_norm(x, w, b, eps))

    dx, dw, db = ops.layer_norm_backward(dy, x, mean, rs, w)
    assert dx.dtype == dtype and dw.dtype == db.dtype == pdtype
    d = dy.double()
    t = d * w.double()
    m1, m2 = t.mean(-1, keepdim=True), (t * xh).mean(-1, keepdim=True)
    dx64 = rstd * (t - m1 - xh * m2)
    # g = dy w rounds once; each of the row's two sums is off by 44 u of its magnitudes and by the error of xh under it; the
    # final expression has four roundings of its terms; rstd's own 25 u multiply the whole
    e = rstd * (64 * U * (t.abs() + t.abs().mean(-1, keepdim=True) + xh.abs() * (t * xh).abs().mean(-1, keepdim=True))
                + xh.abs() * (t.abs() * ex).mean(-1, keepdim=True) + ex * m2.abs())
    e = e + 32 * U * rstd * (t.abs() + m1.abs() + (xh * m2).abs())
    within(dx, dx64, e + half(dtype) * (dx64.abs() + e))
    # sums over rows: at most 200 values one after the other in a lane group and 150 behind that (groups of a workgroup, workgroups)
    n = min(rows, 200) + 150
    dw64, db64 = (d * xh).sum(0), d.sum(0)
    ew = n * U * (d * xh).abs().sum(0) + (d.abs() * ex).sum(0)
    within(dw, dw64, ew + half(pdtype) * (dw64.abs() + ew))
    eb = n * U * d.abs().sum(0)
    within(db, db64, eb + half(pdtype) * (db64.abs() + eb))


@pytest.mark.parametrize("rows,C,dtype", [(100000, 32, BF16), (40000, 128, F32), (70001, 33, BF16), (20000, 512, BF16), (9000, 2048, F32)])
def test_layer_norm_many_rows(rows, C, dtype):
    """Sizes at which every lane group takes several rows and the workspace all its workgroups."""
    g = gen(C)
    x, dy = randn(g, rows, C, dtype=dtype) + 0.5, randn(g, rows, C, dtype=dtype)
    w, b = 1 + 0.3 * randn(g, C), 0.3 * randn(g, C)
    y64, xh, rstd = norm64(x, w, b, 1e-5)
    ex = xh_error(x, xh, rstd)
    y, mean, rs = ops.layer_norm_forward(x, w, b)
    within(y, y64, ex * w.double().abs() + 2 * U * ((xh * w.double()).abs() + b.double().abs()) + half(dtype) * y64.abs() * (1 + 1e-6) + 1e-30)
    dx, dw, db = ops.layer_norm_backward(dy, x, mean, rs, w)
    d = dy.double()
    # rows of one lane group: at most 1024 workgroups of at least 4 groups, but no fewer than 8 rows each
    n = max(8, math.ceil(rows / 1024)) + 200
    ew = n * U * (d * xh).abs().sum(0) + (d.abs() * ex).sum(0)
    within(dw, (d * xh).sum(0), ew + half(F32) * ew + U * (d * xh).sum(0).abs())
    within(db, d.sum(0), n * U * d.abs().sum(0) + U * d.sum(0).abs())
    again = ops.layer_norm_backward(dy, x, mean, rs, w)
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again)), "the same call gives other bits"


def test_layer_norm_gradient_against_differences():
    """dx, dw, db along random directions against central differences of the 64-bit forward pass; the differences' own error is
    what halving the step changes."""
    g = gen(5)
    x, w, b, dy = randn(g, 6, 37), 1 + 0.3 * randn(g, 37), randn(g, 37), randn(g, 6, 37)
    xl, wl, bl = (t.clone().requires_grad_(True) for t in (x, w, b))
    got = torch.autograd.grad(ops.layer_norm(xl, wl, bl), (xl, wl, bl), dy)
    loss = lambda a: (norm64(a[0], a[1], a[2], 1e-5)[0] * dy.double()).sum()
    for k in range(3):
        base = [x.double(), w.double(), b.double()]
        v = randn(g, *base[k].shape).double()

        def slope(h):
            up, dn = list(base), list(base)
            up[k], dn[k] = base[k] + h * v, base[k] - h * v
            return float((loss(up) - loss(dn)) / (2 * h))
        d1, d2 = slope(1e-4), slope(5e-5)
        # the gradient's fp32 entries are off by about 100 u of their terms' magnitude (the bounds of the test above)
        tol = 2 * abs(d1 - d2) + 200 * U * float((got[k].double().abs() + 1).mul(v.abs()).sum()) + 1e-9
        assert abs(float((got[k].double() * v).sum()) - d2) <= tol, (k, d1, d2)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layer_norm_autograd_partial_and_broadcast(dtype):
    g = gen(8)
    x, dy = randn(g, 2, 5, 3, 48, dtype=dtype), randn(g, 2, 5, 3, 48, dtype=dtype)
    w, b = (1 + 0.2 * randn(g, 48)), randn(g, 48, dtype=BF16)
    y, mean, rs = ops.layer_norm_forward(x, w, b)
    full = ops.layer_norm_backward(dy, x, mean, rs, w)
    for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1), (1, 1, 1)):
        xs = x.clone().requires_grad_(bool(need[0]))
        ws, bs = w.clone().requires_grad_(bool(need[1])), b.clone().requires_grad_(bool(need[2]))
        out = ops.layer_norm(xs, ws, bs)
        assert torch.equal(out.detach(), y)
        out.backward(dy)
        for k, (t, f) in enumerate(zip((xs, ws, bs), full)):
            if need[k]:
                assert t.grad.dtype == t.dtype and torch.equal(t.grad, f.to(t.dtype))
            else:
                assert t.grad is None
    # no weight, no bias; a broadcast input and a broadcast output gradient
    one = x[:, :1, :1].clone().requires_grad_(True)
    z = ops.layer_norm(one.expand(2, 5, 3, 48))
    z.sum().backward()
    zz, mm, rr = ops.layer_norm_forward(one.detach().expand(2, 5, 3, 48).contiguous())
    assert torch.equal(z.detach(), zz)
    dx = ops.layer_norm_backward(torch.ones_like(zz), one.detach().expand(2, 5, 3, 48).contiguous(), mm, rr)[0]
    assert torch.equal(one.grad, dx.sum((1, 2), keepdim=True))
    # weight used twice: its gradient is the sum of both
    ws = w.clone().requires_grad_(True)
    (ops.layer_norm(x, ws).float().sum() + ops.layer_norm(x, ws).float().sum()).backward()
    ones = ops.layer_norm_backward(torch.ones_like(y), x, mean, rs, w)[1]
    assert torch.equal(ws.grad, ones + ones)


def test_layer_norm_special_rows():
    """Infinities and NaN stay in their rows; constant and empty rows; a row far from zero."""
    g = gen(3)
    x = randn(g, 7, 40)
    x[1, 3], x[2, 5], x[4] = float("nan"), float("inf"), 2.5
    x[5] += 1000.0
    y = ops.layer_norm(x)
    assert torch.isnan(y[1]).all() and torch.isnan(y[2]).all()
    assert torch.equal(y[4], torch.zeros(40, device=DEV))
    y64, xh, rstd = norm64(x[[0, 3, 5, 6]], None, None, 1e-5)
    within(y[[0, 3, 5, 6]], y64, xh_error(x[[0, 3, 5, 6]], xh, rstd) + 4 * U * y64.abs())
    for shape in ((0, 40), (2, 0, 40)):
        e = torch.empty(shape, device=DEV)
        out, m, r = ops.layer_norm_forward(e)
        assert out.shape == shape and m.shape == shape[:-1]
        w = torch.ones(40, device=DEV, requires_grad=True)
        b = torch.ones(40, device=DEV, requires_grad=True)
        ops.layer_norm(e, w, b).sum().backward()
        assert torch.equal(w.grad, torch.zeros(40, device=DEV)) and torch.equal(b.grad, torch.zeros(40, device=DEV))
        q, s = ops.quantize_rows(e)
        assert q.shape == shape and s.shape == shape[:-1]


# ---- rows in 8 bits -------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,C", SIZES)
def test_quantize_rows(rows, C, dtype):
    """Equal, value by value, to the definition in 64 bits; zeros up to the row's 16-byte border."""
    g = gen(rows * 31 + C)
    x = (randn(g, rows, C) * torch.exp(3 * randn(g, rows, 1))).to(dtype)
    q, s = ops.quantize_rows(x)
    q64, s64 = quant64(x)
    assert torch.equal(s, s64) and torch.equal(q, q64)
    if q.stride(0) != C and rows:
        full = q.as_strided((rows, q.stride(0)), (q.stride(0), 1))
        assert full.shape[1] % 16 == 0 and not full[:, C:].any()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_quantize_rows_borders_and_special_rows(dtype):
    """Values on and next to the borders between two steps, rows of zeros, the smallest and the largest numbers, NaN, infinity."""
    k = torch.arange(-127, 127, device=DEV).double() + 0.5
    rows = [torch.cat([k, k.new_tensor([127.0, -127.0])])]                      # scale 1: every value a tie
    for s in (0.37, 3.0, 1e-30, 1e30, 2.0 ** -126):
        near = torch.cat([k * s, k.new_tensor([127.0 * s, -127.0 * s])])
        rows += [near, near * (1 + 1e-7), near * (1 - 1e-7), near.roll(1) / 3]
    fm = torch.finfo(dtype)
    rows += [torch.zeros(256, device=DEV).double(), torch.full((256,), fm.max, device=DEV).double(),
             torch.full((256,), fm.smallest_normal, device=DEV).double(), torch.full((256,), fm.smallest_normal / 4, device=DEV).double(),
             k.new_tensor([1.49e-36] * 256), k.new_tensor([1.51e-36] * 256)]
    x = torch.stack(rows).to(dtype)
    bad = x[:4].clone()
    bad[0, 0], bad[1, 77], bad[2, 255], bad[3, 3] = float("nan"), float("inf"), float("-inf"), float("nan")
    x = torch.cat([x, bad, x[:3]])
    q, s = ops.quantize_rows(x)
    q64, s64 = quant64(x)
    assert torch.equal(s.nan_to_num(-1), s64.nan_to_num(-1)) and torch.equal(q, q64)
    assert torch.isnan(s[-7:-3]).all() and not q[-7:-3].any()
    y = ops.matmul_i8(q, s, ops.LinearI8.quantize(torch.randn(5, 256, device=DEV)))
    assert torch.isnan(y[-7:-3]).all() and torch.isfinite(y[:1]).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,C", [(1, 1), (3, 7), (64, 24), (17, 255), (400, 512), (31, 1024), (7, 2050), (2, 8192), (30000, 64)])
def test_layer_norm_quantize(rows, C, dtype):
    """The steps of the fused form stand for the norm's values to half a step, and the scale is the row's largest value."""
    g = gen(C * 7 + rows)
    x = randn(g, rows, C, dtype=dtype) * 2 + 0.3
    w, b = 1 + 0.3 * randn(g, C), 0.3 * randn(g, C)
    q, s = ops.layer_norm_quantize(x, w, b)
    y64, xh, rstd = norm64(x, w, b, 1e-5)
    e = (xh_error(x, xh, rstd) * w.double().abs() + 2 * U * ((xh * w.double()).abs() + b.double().abs()))
    top = y64.abs().amax(-1)
    within(s, top / 127, (e.amax(-1) + 2 * U * top) / 127)
    within(q.double() * s.double()[:, None], y64, e + 0.5 * s.double()[:, None] * (1 + 4 * U) + 127 * U * s.double()[:, None])


# ---- product ------------------------------------------------------------------------------------------------------------------
def operands(g, M, K, N, full=False):
    q = torch.randint(-128 if full else -127, 128, (M, K), generator=g, device=DEV, dtype=torch.int8)
    wq = torch.randint(-128 if full else -127, 128, (N, K), generator=g, device=DEV, dtype=torch.int8)
    s, ws = torch.rand(M, generator=g, device=DEV) * 0.01, torch.rand(N, generator=g, device=DEV) * 0.01
    return q, s, wq, ws, randn(g, N)


PRODUCTS = [(1, 1, 1), (1, 64, 16), (2, 1024, 1024), (16, 100, 33), (17, 128, 128), (63, 65, 75), (100, 1000, 255), (128, 128, 128),
            (129, 192, 144), (400, 1024, 512), (1000, 64, 48), (2888, 1000, 255), (4097, 256, 130), (9000, 320, 255), (20000, 48, 512),
            (3000, 4096, 1024), (30001, 16, 24)]


@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("M,K,N", PRODUCTS)
def test_matmul_i8(M, K, N, out):
    g = gen(M + 3 * K + 7 * N)
    q, s, wq, ws, bias = operands(g, M, K, N, full=True)
    res = randn(g, M, N, dtype=out)
    lin, bare = ops.LinearI8(wq, ws, bias), ops.LinearI8(wq, ws)
    for act, mode, r, l in (("none", "after", None, bare), ("silu", "after", res, lin), ("leaky", "before", res, lin), ("silu", "before", None, lin)):
        y = ops.matmul_i8(q, s, l, act=act, slope=0.1, res=r, res_mode=mode, out_dtype=out)
        want, e = product64(q, s, wq, ws, bias if l is lin else None, act, 0.1, r, mode)
        assert y.shape == (M, N) and y.dtype == out
        within(y, want, e + half(out) * (want.abs() + e) + 1e-37)


@pytest.mark.parametrize("K", [131071, 20000])
def test_matmul_i8_longest_sums(K):
    """The largest sums a 32-bit integer has to hold."""
    q = torch.full((3, K), -128, device=DEV, dtype=torch.int8)
    q[1] = 127
    wq = torch.full((20, K), -128, device=DEV, dtype=torch.int8)
    wq[7:] = 127
    s, ws = torch.ones(3, device=DEV), torch.ones(20, device=DEV)
    y = ops.matmul_i8(q, s, ops.LinearI8(wq, ws), out_dtype=F32)
    want = q.cpu().double() @ wq.cpu().double().t()
    assert torch.equal(y.cpu(), want.float())


@pytest.mark.parametrize("out", [F32, BF16])
def test_matmul_i8_does_not_depend_on_the_batch(out):
    """Whichever kernel takes the rows: a row's result is the same alone, among few and among many."""
    g = gen(77)
    q, s, wq, ws, bias = operands(g, 40000, 512, 256)
    lin = ops.LinearI8(wq, ws, bias)
    y = ops.matmul_i8(q, s, lin, act="silu", out_dtype=out)
    for n in (1, 16, 17, 300, 1000, 5000, 20000):
        assert torch.equal(ops.matmul_i8(q[:n], s[:n], lin, act="silu", out_dtype=out), y[:n])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,K,N", [(1, 1, 1), (1, 1024, 1024), (5, 77, 33), (16, 2048, 512), (17, 2049, 75), (100, 1000, 255), (400, 1024, 512),
                                   (200, 100, 1000), (169, 384, 1536), (300, 1025, 256), (33, 8192, 64), (3000, 200, 130)])
def test_linear_i8_is_quantisation_and_product(M, K, N, dtype):
    """In one launch or two: the bits of quantize_rows followed by matmul_i8, rows without a scale and rows of zeros among them."""
    g = gen(M + 3 * K + 7 * N)
    x = (randn(g, M, K) * torch.exp(2 * randn(g, M, 1))).to(dtype)
    x[M // 2] = 0
    if M > 4:
        x[1, K // 2], x[3, 0] = float("nan"), float("-inf")
        x[4] = torch.where(torch.arange(K, device=DEV) % 2 == 0, 1.0, -0.5).to(dtype)        # every other value on a border
    lin = ops.LinearI8.quantize(randn(g, N, K), randn(g, N))
    wide = torch.zeros(M, K + 5, device=DEV, dtype=dtype)
    wide[:, 3:K + 3] = x
    for out in (F32, BF16):
        res = randn(g, M, N, dtype=out)
        q, s = ops.quantize_rows(x)
        for kw in (dict(), dict(act="silu", res=res), dict(act="leaky", res=res, res_mode="before")):
            want = ops.matmul_i8(q, s, lin, out_dtype=out, **kw)
            for t in (x, wide[:, 3:K + 3]):
                got = ops.linear_i8(t, lin, out_dtype=out, **kw)
                assert torch.equal(got.nan_to_num(12345.0), want.nan_to_num(12345.0)) and torch.equal(got.isnan(), want.isnan())
    if M > 4:
        assert want[1].isnan().all() and want[3].isnan().all() and torch.isfinite(want[2]).all()


def test_rows_at_any_distance_and_address():
    """Channel slices of wider maps, odd pitches and addresses, transposed and broadcast maps."""
    g = gen(21)
    for dtype in (F32, BF16):
        big = randn(g, 3, 10, 11, 70, dtype=dtype)
        w, b = randn(g, 64), randn(g, 64)
        for x in (big[..., :64], big[..., 1:65], big[..., 6:70], big[:, 1:9, 2:7, 3:67], big[..., :64].transpose(0, 1), big[0, 0, 0, :64],
                  big[:, :1, :, :64].expand(3, 10, 11, 64), big[:, :, :, :64][:, ::2]):
            ref = x.contiguous().clone()
            assert torch.equal(ops.layer_norm(x, w, b), ops.layer_norm(ref, w, b))
            for a, c in zip(ops.quantize_rows(x) + ops.layer_norm_quantize(x, w, b), ops.quantize_rows(ref) + ops.layer_norm_quantize(ref, w, b)):
                assert torch.equal(a, c)
            y, m, r = ops.layer_norm_forward(ref, w, b)
            dy = randn(g, *ref.shape, dtype=dtype)
            wide = torch.zeros(*ref.shape[:-1], 71, device=DEV, dtype=dtype)
            wide[..., 5:69] = dy
            for a, c in zip(ops.layer_norm_backward(wide[..., 5:69], x, m, r, w), ops.layer_norm_backward(dy, ref, m, r, w)):
                assert torch.equal(a, c)
    # 8-bit rows: any pitch and address, the last row at the very end of its memory
    q, s, wq, ws, bias = operands(g, 200, 77, 40)
    lin = ops.LinearI8(wq, ws, bias)
    want = ops.matmul_i8(q, s, lin)
    for pitch, off in ((77, 0), (80, 0), (80, 3), (96, 16), (101, 5), (128, 32)):
        flat = torch.randint(-127, 128, (199 * pitch + off + 77,), generator=g, device=DEV, dtype=torch.int8)
        v = flat.as_strided((200, 77), (pitch, 1), off)
        v.copy_(q)
        assert torch.equal(ops.matmul_i8(v, s, lin), want), (pitch, off)
    wide = torch.zeros(200, 60, device=DEV)
    r = randn(g, 200, 40)
    wide[:, 3:43] = r
    assert torch.equal(ops.matmul_i8(q, s, lin, res=wide[:, 3:43], out_dtype=F32), ops.matmul_i8(q, s, lin, res=r, out_dtype=F32))


def test_rows_beyond_32_bit_offsets():
    """Maps whose last rows lie more than 2^32 bytes and 2^31 values behind the first."""
    rows, ld = 70001, 40000
    big = torch.empty(rows, ld, device=DEV, dtype=BF16)            # 5.6 GB, touched in a few columns
    x = big[:, 64:128]
    g = gen(1)
    x.copy_(randn(g, rows, 64))
    ref = x.contiguous()
    assert torch.equal(ops.layer_norm(x), ops.layer_norm(ref))
    q, s = ops.quantize_rows(x)
    q2, s2 = ops.quantize_rows(ref)
    assert torch.equal(q, q2) and torch.equal(s, s2)
    lin = ops.LinearI8.quantize(randn(g, 48, 64))
    want = ops.matmul_i8(q, s, lin)
    wide8 = big.view(torch.int8)[:, 16:80]                         # 8-bit rows 80 000 bytes apart
    wide8.copy_(q)
    assert torch.equal(ops.matmul_i8(wide8, s, lin), want)
    # the library's own slices: output rows that far apart
    d = _ffi.MatmulI8Desc(q.data_ptr(), s.data_ptr(), lin.w.data_ptr(), lin.scale.data_ptr(), None, None, big.data_ptr(), rows, 64, 48,
                          lin.kp, lin.n_pad, 64, 0, ld, 1024, 0, 0, 0, 0.0, 0, _ffi.BF16)
    _ffi.check(_ffi.lib().ydet_matmul_i8(d, None, 0, _ffi.current_stream()))
    assert torch.equal(big[:, 1024:1072], want)


def test_a_token_wise_block():
    """norm -> 8 bits -> 256 channels, SiLU -> 8 bits -> 64 channels + shortcut, as a network runs it: every product within its
    bound of the 64-bit one on the rows it was given, and the whole near the floating block."""
    g = gen(12)
    N, H, W, C = 2, 13, 13, 64
    x = randn(g, N, H, W, C, dtype=BF16)
    w, b = 1 + 0.2 * randn(g, C), 0.1 * randn(g, C)
    w1, w2 = randn(g, 256, C) / 8, randn(g, C, 256) / 16
    l1, l2 = ops.LinearI8.quantize(w1, randn(g, 256)), ops.LinearI8.quantize(w2[:, :, None, None])
    q, s = ops.layer_norm_quantize(x, w, b)
    h = ops.matmul_i8(q, s, l1, act="silu")
    y = ops.linear_i8(h, l2, res=x)
    assert h.shape == (N, H, W, 256) and y.shape == x.shape and y.dtype == BF16
    want, e = product64(q, s, l1.w[:256, :C], l1.scale[:256], l1.bias[:256], "silu", 0.1, None, "after")
    within(h, want, e + half(BF16) * (want.abs() + e))
    q2, s2 = ops.quantize_rows(h)
    want, e = product64(q2, s2, l2.w[:C, :256], l2.scale[:C], None, "none", 0.1, x, "after")
    within(y, want, e + half(BF16) * (want.abs() + e))
    # the floating block: 8 bits put noise of uniform half steps on rows and weights, amax / 127 / sqrt(12) each per value
    z = norm64(x, w, b, 1e-5)[0]
    hz = z @ w1.double().t() + l1.bias[:256].double()
    hz = hz * torch.sigmoid(hz)
    yz = hz @ w2.double().t() + x.double()
    assert float((y.double() - yz).norm() / (yz - x.double()).norm()) < 0.05


# ---- streams, graphs -------------------------------------------------------------------------------------------------------
def test_streams_and_graph_replays():
    """A block captured into a graph: every replay, with eager work and synchronisations between, equals the eager result; two
    streams at once give what one gives."""
    g = gen(14)
    x, dy = randn(g, 4097, 96, dtype=BF16), randn(g, 4097, 96, dtype=BF16)
    w, b = 1 + 0.2 * randn(g, 96), randn(g, 96)
    lin = ops.LinearI8.quantize(randn(g, 128, 96))

    def block(x, dy):
        y, m, r = ops.layer_norm_forward(x, w, b)
        grads = ops.layer_norm_backward(dy, x, m, r, w)
        q, s = ops.layer_norm_quantize(x, w, b)
        return (y,) + grads + (ops.matmul_i8(q, s, lin, act="silu"), ops.linear_i8(x[:7], lin), ops.linear_i8(x, lin, out_dtype=F32))
    sx, sdy = x.clone(), dy.clone()
    block(sx, sdy)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block(sx, sdy)
    second = torch.cuda.CUDAGraph()
    with torch.cuda.graph(second):
        out2 = block(sx, sdy)
    for k in range(4):
        sx.copy_(x * (k + 1))
        sdy.copy_(dy.roll(k, 0))
        want = block(sx.clone(), sdy.clone())
        graph.replay()
        second.replay()
        torch.cuda.synchronize()
        for a, c, e in zip(out, want, out2):
            assert torch.equal(a, c) and torch.equal(e, c)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    want = [block(x * k, dy) for k in (1, 2)]
    torch.cuda.synchronize()
    ins = [x * 1, x * 2]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(5):
        for k, st in enumerate((s1, s2)):
            with torch.cuda.stream(st):
                got[k] = block(ins[k], dy)
    torch.cuda.synchronize()
    for a, c in zip(got, want):
        assert all(torch.equal(p, r) for p, r in zip(a, c))


def test_layer_norm_refuses_to_record_in_a_capture():
    x = torch.randn(8, 16, device=DEV, requires_grad=True)
    ops.layer_norm(x)
    s = torch.zeros(1, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.add_(1)
        with pytest.raises(RuntimeError, match="during graph capture"):
            ops.layer_norm(x)
        with torch.no_grad():
            y = ops.layer_norm(x)
    graph.replay()
    assert torch.equal(y, ops.layer_norm(x).detach())


# ---- refusals ---------------------------------------------------------------------------------------------------------------
def test_refusals():
    x = torch.randn(4, 32, device=DEV)
    lin = ops.LinearI8.quantize(torch.randn(8, 32, device=DEV))
    q, s = ops.quantize_rows(x)
    y, m, r = ops.layer_norm_forward(x)
    for call, err in (
            (lambda: ops.layer_norm(x.half()), TypeError), (lambda: ops.layer_norm(x.cpu()), RuntimeError),
            (lambda: ops.layer_norm(x, torch.ones(31, device=DEV)), ValueError), (lambda: ops.layer_norm(x, torch.ones(32)), RuntimeError),
            (lambda: ops.layer_norm(torch.randn(2, 8193, device=DEV)), RuntimeError), (lambda: ops.layer_norm(x, eps=-1.0), RuntimeError),
            (lambda: ops.layer_norm(torch.randn(3, 0, device=DEV)), ValueError), (lambda: ops.layer_norm(torch.tensor(1.0, device=DEV)), ValueError),
            (lambda: ops.layer_norm_backward(x.bfloat16(), x, m, r), ValueError), (lambda: ops.layer_norm_backward(x[:3], x, m, r), ValueError),
            (lambda: ops.layer_norm_backward(x, x, m[:2], r), ValueError), (lambda: ops.quantize_rows(x.double()), TypeError),
            (lambda: ops.matmul_i8(q, s, lin, act="relu6"), ValueError), (lambda: ops.matmul_i8(q[:, :16], s, lin), ValueError),
            (lambda: ops.matmul_i8(q, s[:2], lin), ValueError), (lambda: ops.matmul_i8(q, s, lin, out_dtype=torch.float16), TypeError),
            (lambda: ops.matmul_i8(q, s, lin, res=torch.zeros(4, 8, device=DEV)), ValueError), (lambda: ops.matmul_i8(x, s, lin), ValueError),
            (lambda: ops.matmul_i8(q, s, lin, res=torch.zeros(4, 7, device=DEV, dtype=BF16)), ValueError),
            (lambda: ops.linear_i8(x[:, :16], lin), ValueError), (lambda: ops.LinearI8(q, s.cpu()), RuntimeError),
            (lambda: ops.LinearI8(q, s[:3]), ValueError), (lambda: ops.LinearI8.quantize(torch.randn(4, 4, 3, 3, device=DEV)), ValueError)):
        with pytest.raises(err):
            call()


# ---- in the planner -----------------------------------------------------------------------------------------------------------
@pytest.fixture
def pointwise_int8():
    engine.set_pointwise_int8(True)
    try:
        yield
    finally:
        engine.set_pointwise_int8(False)
        engine.set_compute_dtype(None)


def _slice(arena, t):
    root, off = t.resolve()
    return arena[root][..., off:off + t.C]


def _overlap(a, b):
    (ra, oa), (rb, ob) = a.resolve(), b.resolve()
    return ra is rb and oa < ob + b.C and ob < oa + a.C


def _intact(opslist, i):
    """Whether the maps of op i still hold what it read and wrote: not external, not worked on in place by it or a later op."""
    a = opslist[i][1]
    mine = [t for t in (a["x"], a["y"], a["res"]) if t is not None]
    return (not any(t.resolve()[0].external for t in mine) and not any(_overlap(t, a["y"]) for t in mine if t is not a["y"])
            and not any(_overlap(t, w) for _, later in opslist[i + 1:] for w in (later.get("y"), later.get("y2")) if w is not None for t in mine))


def _check_products(plan):
    """Every 8-bit convolution of a plan that ran and whose maps are intact: its output equals linear_i8 of its input, bit for bit."""
    seen = 0
    for arena in plan.arenas:
        for i, (kind, a) in enumerate(plan.g.ops):
            if kind != "linear_i8" or not _intact(plan.g.ops, i):
                continue
            act = {_ffi.ACT_NONE: "none", _ffi.ACT_LEAKY: "leaky", _ffi.ACT_SILU: "silu"}[a["act"]]
            res = None if a["res"] is None else _slice(arena, a["res"])
            want = ops.linear_i8(_slice(arena, a["x"]), a["lin"], act, a["slope"], res, "before" if a["res_mode"] == _ffi.RES_BEFORE_ACT else "after",
                                 BF16)
            assert torch.equal(_slice(arena, a["y"]), want)
            seen += 1
    return seen


def test_plan_layers_in_8_bits(pointwise_int8):
    """1x1 layers with SiLU / leaky / no activation, residual after and before it, into and out of concat buffers, and a layer
    norm between them; against the operators and against the bf16 plan."""
    from yolo_amd.synthetic import init_deterministic
    from yolo_amd.yolov5_official.modules import Conv

    class Net(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.a, self.b, self.c = Conv(512, 512), Conv(512, 512), torch.nn.Conv2d(1024, 512, 1)
            self.n, self.d = torch.nn.LayerNorm(1024), Conv(512, 1024, act=False)

        def lower(self, g, x):
            a = self.a.lower(g, x)
            b = self.b.lower(g, a, res=x)
            c = g.conv(g.cat([a, b]), self.c, act=_ffi.ACT_LEAKY, slope=0.1, res=x, res_mode=_ffi.RES_BEFORE_ACT)
            return g.layer_norm(self.d.lower(g, c), self.n)

        def forward(self, x):
            a = self.a(x)
            b = x + self.b(a)
            c = torch.nn.functional.leaky_relu(self.c(torch.cat([a, b], 1)) + x, 0.1)
            return self.n(self.d(c).permute(0, 2, 3, 1)).permute(0, 3, 1, 2)

    net = Net()
    init_deterministic(net, seed=3)
    net = net.to(DEV).eval()
    with torch.no_grad():
        net.n.weight.uniform_(0.5, 1.5)
        net.n.bias.normal_()
    x = randn(gen(2), 2, 512, 13, 11)
    outs = {}
    for on in (True, False):
        engine.set_pointwise_int8(on)
        g = engine.Graph(DEV, "bf16")
        g.to_nchw(net.lower(g, g.input_nchw(*x.shape)), "y")
        plan = g.finalize()
        outs[on] = plan.run(x)["y"].float()
        kinds = [k for k, _ in g.ops]
        assert kinds.count("linear_i8") == (4 if on else 0) and kinds.count("layernorm") == 1 and "copy" not in kinds
        assert _check_products(plan) == (4 if on else 0)
        (nk, na), = [(k, a) for k, a in g.ops if k == "layernorm"]
        assert torch.equal(_slice(plan.arenas[0], na["y"]), ops.layer_norm(_slice(plan.arenas[0], na["x"]), net.n.weight, net.n.bias, net.n.eps))
        assert torch.equal(plan.run(x)["y"].float(), outs[on])
    with torch.no_grad():
        ref = net(x)
    # bf16: every stored value is off by up to 2^-8 of itself, five maps deep, and so are the weights; 8 bits add steps of amax / 127
    # (amax about 4.5 sigma: 1 % of a row's norm) four times to rows and weights
    rel = lambda a: float((a - ref).norm() / ref.norm())
    assert rel(outs[False]) < 5 * 2 * 2.0 ** -8 and rel(outs[True]) < 4 * 2 * 0.0125 + 5 * 2 * 2.0 ** -8


def test_plan_layer_norm_fp32_and_refusal():
    g = engine.Graph(DEV, "fp32")
    n = torch.nn.LayerNorm(24, elementwise_affine=False).to(DEV)
    x = randn(gen(4), 3, 24, 5, 7)
    t = g.input_nchw(*x.shape)
    with pytest.raises(NotImplementedError):
        g.layer_norm(t, torch.nn.LayerNorm(12))
    g.to_nchw(g.layer_norm(t, n), "y")
    y = g.finalize().run(x)["y"]
    assert torch.equal(y, ops.layer_norm(x.permute(0, 2, 3, 1)).permute(0, 3, 1, 2))


@pytest.mark.parametrize("tag,size,batch", [("v3spp", 128, 1), ("v4", 128, 2)])
def test_detector_in_8_bits(pointwise_int8, tag, size, batch):
    """A whole detector with its 1x1 layers in 8 bits: every product checked against the operator on the plan's own maps; switching
    the option off again gives the bf16 result of before."""
    from helpers import build_fa
    from yolo_amd.synthetic import images
    engine.set_compute_dtype("bf16")
    net = build_fa(tag, size).to(DEV)
    x = images(batch, size, seed=1).to(DEV)
    engine.set_pointwise_int8(False)
    with torch.no_grad():
        before = net(x)
        engine.set_pointwise_int8(True)
        net(x)
        plans = [p for p in net._plans().plans.values() if any(k == "linear_i8" for k, _ in p.g.ops)]
        torch.cuda.synchronize()
        assert len(plans) == 1 and _check_products(plans[0]) >= 5
        engine.set_pointwise_int8(False)
        after = net(x)
    for a, b in zip(before, after):
        assert (a == b).all()


def test_plan_in_8_bits_replicas_and_graph(pointwise_int8):
    """Two side-by-side launch lists have workspaces of their own; a plan captured into a graph replays like its eager run."""
    from yolo_amd.synthetic import init_deterministic
    from yolo_amd.yolov5_official.modules import Conv
    net = torch.nn.Sequential(Conv(512, 1024), Conv(1024, 512))
    init_deterministic(net, seed=3)
    net = net.to(DEV).eval()
    x = randn(gen(2), 16, 512, 9, 9)

    def build(n):
        g = engine.Graph(DEV, "bf16")
        g.to_nchw(engine.lower_any(g, net, g.input_nchw(n, 512, 9, 9)), "y")
        return g
    one, two = build(16).finalize(), build(8).finalize(2)
    assert len(two.i8_ws) == 2 and two.i8_ws[0].data_ptr() != two.i8_ws[1].data_ptr()
    want = one.run(x)["y"]
    for _ in range(3):
        assert torch.equal(two.run(x)["y"], want)
    assert _check_products(two) == 4
    replay = engine.GraphReplay(lambda t: one.run(t)["y"])
    for k in range(4):
        xk = x * (k + 1)
        want = one.run(xk)["y"].clone()
        assert torch.equal(replay(xk), want)
        torch.cuda.synchronize()


# ---- calls at the edges -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("M,K,N,dtype", [(5, 64, 32, BF16), (3000, 200, 130, F32)])
def test_norm_and_product_in_one_call_of_the_library(M, K, N, dtype):
    g = gen(K)
    x, w, b = randn(g, M, K, dtype=dtype), 1 + 0.3 * randn(g, K), randn(g, K)
    lin = ops.LinearI8.quantize(randn(g, N, K), randn(g, N))
    want = ops.matmul_i8(*ops.layer_norm_quantize(x, w, b), lin, act="silu", out_dtype=F32)
    y = torch.empty(M, N, device=DEV)
    q = _ffi.QuantizeDesc(x.data_ptr(), None, None, w.data_ptr(), b.data_ptr(), M, K, K, 0, 0, ops._dt(x), _ffi.F32, 1, 1e-5)
    d = _ffi.MatmulI8Desc(None, None, lin.w.data_ptr(), lin.scale.data_ptr(), lin.bias.data_ptr(), None, y.data_ptr(), M, K, N, lin.kp, lin.n_pad,
                          0, 0, N, 0, 0, 0, _ffi.ACT_SILU, 0.0, 0, _ffi.F32)
    lib = _ffi.lib()
    n = lib.ydet_linear_i8_workspace_bytes(q, d)
    ws = torch.empty(n, device=DEV, dtype=torch.uint8)
    _ffi.check(lib.ydet_linear_i8(q, d, ws.data_ptr(), n, _ffi.current_stream()))
    assert n > 0 and torch.equal(y, want)


@pytest.mark.parametrize("wdt,bdt", [(BF16, F32), (F32, BF16)])
def test_gradients_of_parameters_of_two_types(wdt, bdt):
    # either gradient is rounded to its own parameter's type alone
    rows, C = 300, 96
    g = gen(7)
    x, dy = randn(g, rows, C), randn(g, rows, C)
    w, b = (1 + 0.3 * randn(g, C)).to(wdt).requires_grad_(), randn(g, C).to(bdt).requires_grad_()
    ops.layer_norm(x, w, b).backward(dy)
    xd, dyd = x.double(), dy.double()
    xh = (xd - xd.mean(-1, keepdim=True)) / (xd.var(-1, keepdim=True, unbiased=False) + 1e-5).sqrt()
    for got, terms, size, dt in ((w.grad, dyd * xh, dyd.abs() * (xh.abs() + 2 * xd.abs() + 1), wdt), (b.grad, dyd, dyd.abs(), bdt)):
        assert got.dtype == dt
        want = terms.sum(0)
        # fp32 sums of `rows` terms, no chain of additions longer than their number; x-hat is off by a few steps of itself (the
        # deviation) and of |x| and the mean (|mean| < 1/2, 1 / deviation < 2); then one rounding to the parameter's type
        tol = (rows + 16) * 2.0 ** -24 * size.sum(0) + (2.0 ** -8 * want.abs() if dt is BF16 else 0)
        assert ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("M,K,N", [(3, 64, 40), (900, 130, 40), (257, 64, 1000), (6400, 1030, 520), (23104, 2050, 500)])
def test_weights_padded_further_than_needed(M, K, N):
    # zeros behind K up to a pitch of the caller's choice; the rows of x end with their memory
    g = gen(M)
    q, s, wq, ws, bias = operands(g, M, K, N)
    lin = ops.LinearI8(wq, ws, bias)
    want = ops.matmul_i8(q, s, lin)
    lin.kp += 448
    wide = torch.zeros(lin.n_pad, lin.kp, device=DEV, dtype=torch.int8)
    wide[:N, :K] = wq
    lin.w = wide
    assert torch.equal(ops.matmul_i8(q, s, lin), want)
    x = randn(g, M, K)
    assert torch.equal(ops.linear_i8(x, lin), ops.matmul_i8(*ops.quantize_rows(x), lin, out_dtype=F32))


@pytest.mark.parametrize("M,K,N", [(900, 77, 40), (700, 1000, 255), (3000, 1001, 130), (6400, 1030, 520), (23104, 2050, 500), (40000, 66, 64)])
def test_rows_at_any_word(M, K, N):
    """8-bit rows at 4-byte addresses and pitches, the last one at the very end of its memory (every tile, with and without a
    whole word at the rows' end); the values between the rows do not matter."""
    g = gen(M + K)
    q, s, wq, ws, bias = operands(g, M, K, N)
    lin = ops.LinearI8(wq, ws, bias)
    want, e = product64(q, s, wq, ws, bias, "none", 0.1, None, "after")
    k4 = (K + 3) // 4 * 4
    for pitch, off in ((k4, 0), (k4 + 4, 4), (k4 + 44, 12), (K, 0), (K, 1)):
        flat = torch.randint(-127, 128, ((M - 1) * pitch + off + K,), generator=g, device=DEV, dtype=torch.int8)
        v = flat.as_strided((M, K), (pitch, 1), off)
        v.copy_(q)
        within(ops.matmul_i8(v, s, lin, out_dtype=F32), want, e + half(F32) * (want.abs() + e) + 1e-37)


def test_second_derivative_is_an_error():
    x = torch.randn(4, 24, device=DEV, requires_grad=True)
    w = torch.randn(24, device=DEV, requires_grad=True)
    gx, = torch.autograd.grad(ops.layer_norm(x, w).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        gx.sum().backward()
    gx, = torch.autograd.grad(ops.layer_norm(x, w).square().sum(), x)
    assert not gx.requires_grad


def test_input_changed_behind_the_forward_pass_is_an_error():
    x = torch.randn(4, 24, device=DEV)
    w = torch.randn(24, device=DEV, requires_grad=True)
    y = ops.layer_norm(x, w)
    x.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_products_without_rows_and_single_rows():
    lin = ops.LinearI8.quantize(torch.randn(20, 30, device=DEV))
    for lead in ((0,), (3, 0), (0, 5)):
        q, s = ops.quantize_rows(torch.empty(*lead, 30, device=DEV))
        assert ops.matmul_i8(q, s, lin).shape == lead + (20,)
        assert ops.linear_i8(torch.empty(*lead, 30, device=DEV), lin, res=torch.empty(*lead, 20, device=DEV)).shape == lead + (20,)
    x = torch.randn(30, device=DEV)
    q, s = ops.quantize_rows(x)
    assert q.shape == (30,) and s.shape == ()
    y = ops.matmul_i8(q, s, lin, out_dtype=F32)
    assert y.shape == (20,) and torch.equal(y, ops.linear_i8(x, lin)) and torch.equal(y, ops.linear_i8(x[None, None], lin)[0, 0])
    y, m, r = ops.layer_norm_forward(x)
    assert y.shape == (30,) and m.shape == r.shape == ()
    assert torch.equal(ops.layer_norm_backward(y, x, m, r)[0], ops.layer_norm_backward(y[None], x[None], m[None], r[None])[0][0])


@pytest.mark.parametrize("M", [65, 127, 129, 191, 193, 255, 257, 321])
def test_tails_of_every_tile(M):
    """The last rows of a tile, the scales behind them and the last channels, for K on both sides of the kernels' choices."""
    g = gen(M)
    for reps, K, N in ((1, 2048, 8), (40, 1024, 320), (130, 2050, 1100), (100, 130, 520), (300, 64, 72)):
        rows = M * reps + M % 7
        q, s, wq, ws, bias = operands(g, rows, K, N)
        lin = ops.LinearI8(wq, ws, bias)
        y = ops.matmul_i8(q, s, lin, act="leaky", out_dtype=F32)
        # (the last rows and a few others: the whole product in 64 bits would take long)
        some = torch.cat([torch.arange(0, rows, max(1, rows // 50), device=DEV), torch.arange(max(0, rows - 200), rows, device=DEV)])
        want, e = product64(q[some], s[some], wq, ws, bias, "leaky", 0.1, None, "after")
        within(y[some], want, e + half(F32) * (want.abs() + e) + 1e-37)


def test_outputs_leave_the_rest_alone():
    """Output slices of wider maps, through the library: the channels beside and the rows behind them stay as they were."""
    g = gen(9)
    lib, st = _ffi.lib(), _ffi.current_stream()
    for rows, K, N, coff in ((5, 77, 30, 3), (700, 128, 72, 8), (40000, 64, 64, 1), (7000, 1024, 200, 5)):
        ld = N + coff + 7
        q, s, wq, ws, bias = operands(g, rows, K, N)
        lin = ops.LinearI8(wq, ws, bias)
        q, s = ops.quantize_rows(q.float() * s[:, None])
        want = ops.matmul_i8(q, s, lin, out_dtype=F32)
        buf = torch.full((rows + 9, ld), -7.0, device=DEV)
        d = _ffi.MatmulI8Desc(q.data_ptr(), s.data_ptr(), lin.w.data_ptr(), lin.scale.data_ptr(), lin.bias.data_ptr(), None, buf.data_ptr(), rows, K,
                              N, lin.kp, lin.n_pad, q.stride(0), 0, ld, coff, 0, 0, 0, 0.0, 0, _ffi.F32)
        _ffi.check(lib.ydet_matmul_i8(d, None, 0, st))
        assert torch.equal(buf[:rows, coff:coff + N], want)
        buf[:rows, coff:coff + N] = -7.0
        assert (buf == -7.0).all()
    for C, dtype in ((30, F32), (30, BF16), (512, BF16), (2049, F32)):
        x = randn(g, 50, C, dtype=dtype)
        want = ops.layer_norm(x)
        buf = torch.full((53, C + 9), -7.0, device=DEV, dtype=dtype)
        d = _ffi.LayerNormDesc(x.data_ptr(), buf.data_ptr(), None, None, None, None, 50, C, C, 0, C + 9, 4, ops._dt(x), 0, 1e-5)
        _ffi.check(lib.ydet_layer_norm(d, st))
        assert torch.equal(buf[:50, 4:C + 4], want)
        buf[:50, 4:C + 4] = -7.0
        assert (buf == -7.0).all()
        Cp = (C + 15) // 16 * 16
        qb = torch.full((53, Cp + 16), -7, device=DEV, dtype=torch.int8)
        sb = torch.full((53,), -7.0, device=DEV)
        d = _ffi.QuantizeDesc(x.data_ptr(), qb.data_ptr(), sb.data_ptr(), None, None, 50, C, C, 0, Cp + 16, ops._dt(x), 0, 0, 0.0)
        _ffi.check(lib.ydet_quantize_rows_i8(d, st))
        q, s = ops.quantize_rows(x)
        assert torch.equal(qb[:50, :C], q) and torch.equal(sb[:50], s) and not qb[:50, C:Cp].any()
        assert (qb[:, Cp:] == -7).all() and (qb[50:] == -7).all() and (sb[50:] == -7).all()


def test_in_place():
    """y may be x, dx may be dy, and a product's output its residual."""
    g = gen(10)
    x, dy = randn(g, 900, 40, dtype=BF16), randn(g, 900, 40, dtype=BF16)
    lib, st = _ffi.lib(), _ffi.current_stream()
    y, m, r = ops.layer_norm_forward(x)
    dx, _, _ = ops.layer_norm_backward(dy, x, m, r, need=(True, False, False))
    d2 = dy.clone()
    d = _ffi.LayerNormGradDesc(d2.data_ptr(), x.data_ptr(), d2.data_ptr(), None, m.data_ptr(), r.data_ptr(), None, None, 900, 40, 40, 0, 40, 0, 40, 0,
                               _ffi.BF16, 0)
    _ffi.check(lib.ydet_layer_norm_backward(d, None, 0, st))
    assert torch.equal(d2, dx)
    x2 = x.clone()
    _ffi.check(lib.ydet_layer_norm(_ffi.LayerNormDesc(x2.data_ptr(), x2.data_ptr(), None, None, None, None, 900, 40, 40, 0, 40, 0, _ffi.BF16, 0, 1e-5), st))
    assert torch.equal(x2, y)
    lin = ops.LinearI8.quantize(randn(g, 40, 40))
    q, s = ops.quantize_rows(x)
    want = ops.matmul_i8(q, s, lin, act="silu", res=x)
    x3 = x.clone()
    d = _ffi.MatmulI8Desc(q.data_ptr(), s.data_ptr(), lin.w.data_ptr(), lin.scale.data_ptr(), None, x3.data_ptr(), x3.data_ptr(), 900, 40, 40, lin.kp,
                          lin.n_pad, q.stride(0), 0, 40, 0, 40, 0, _ffi.ACT_SILU, 0.0, _ffi.RES_AFTER_ACT, _ffi.BF16)
    _ffi.check(lib.ydet_matmul_i8(d, None, 0, st))
    assert torch.equal(x3, want)


@pytest.mark.parametrize("K", [30, 32, 64])
@pytest.mark.parametrize("lead", [(0,), (3, 0), (0, 5)])
def test_empty_batches_through_a_block(lead, K):
    """Norm, 8 bits and products of a batch without rows, at row pitches that are and are not multiples of 4."""
    lin = ops.LinearI8.quantize(torch.randn(20, K, device=DEV))
    x = torch.empty(*lead, K, device=DEV, dtype=BF16)
    q, s = ops.layer_norm_quantize(x, torch.ones(K, device=DEV))
    assert q.shape == lead + (K,) and s.shape == lead
    y = ops.matmul_i8(q, s, lin, act="silu", res=torch.empty(*lead, 20, device=DEV, dtype=BF16))
    assert y.shape == lead + (20,) and y.dtype == BF16
    assert ops.matmul_i8(*ops.quantize_rows(x), lin, out_dtype=F32).shape == ops.linear_i8(x, lin).shape == lead + (20,)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,K,N", [(1, 64, 64), (40, 512, 512), (100, 256, 256), (33, 200, 90), (900, 128, 128), (5000, 96, 96)])
def test_linear_in_place(M, K, N, dtype):
    """The output over the floating rows it is made from (and over the residual), few rows and many: the bits of the call apart,
    given a workspace; few rows without one are refused."""
    g = gen(M + K)
    lib, st = _ffi.lib(), _ffi.current_stream()
    x = randn(g, M, K, dtype=dtype)
    lin = ops.LinearI8.quantize(randn(g, N, K) / math.sqrt(K), randn(g, N))
    shortcut = N == K
    want = ops.linear_i8(x, lin, act="silu", res=x if shortcut else None)
    dt = ops._dt(x)
    at = x.clone()
    q = _ffi.QuantizeDesc(at.data_ptr(), None, None, None, None, M, K, K, 0, 0, dt, _ffi.F32, 0, 0.0)
    d = _ffi.MatmulI8Desc(None, None, lin.w.data_ptr(), lin.scale.data_ptr(), lin.bias.data_ptr(), at.data_ptr(), at.data_ptr(), M, K, N, lin.kp,
                          lin.n_pad, 0, 0, K, 0, K, 0, _ffi.ACT_SILU, 0.0, _ffi.RES_AFTER_ACT if shortcut else _ffi.RES_NONE, dt)
    assert lib.ydet_linear_i8(q, d, None, 0, st) < 0
    nbytes = M * ((K + 15) // 16 * 16) + (M + 3) // 4 * 16
    ws = torch.empty(nbytes, device=DEV, dtype=torch.uint8)
    _ffi.check(lib.ydet_linear_i8(q, d, ws.data_ptr(), nbytes, st))
    assert torch.equal(at[:, :N], want) and torch.equal(at[:, N:], x[:, N:])


def test_parameter_gradients_of_very_many_rows():
    """The sums over rows keep their error however many there are: a lane adds at most 1024 rows one after the other, then come the
    64 groups of a workgroup, 11 launches and a tree of 16.  (Equal terms of this value drift one way: a chain of all the rows of a
    lane group, 10 681, ends 1.5e-4 off.)"""
    rows, c = 700_000_001, 1.521
    dy = torch.full((rows, 1), c, device=DEV)
    x = torch.ones(rows, 1, device=DEV)
    mean, rstd = torch.zeros(rows, device=DEV), torch.ones(rows, device=DEV)
    _, dw, db = ops.layer_norm_backward(dy, x, mean, rstd, need=(False, True, True))
    want = rows * float(torch.tensor(c, dtype=F32))
    for got in (dw, db):
        assert abs(float(got) - want) <= (1024 + 64 + 11 + 16) * U * want
    # and every row is there once: rows and launches of unlike values
    dy[:] = 0
    marks = torch.tensor([0, 1, 63, 67_108_863, 67_108_864, 134_217_727, 500_000_000, rows - 1], device=DEV)
    dy[marks, 0] = 2.0 ** torch.arange(8, device=DEV)
    x[marks, 0] = 3.0
    dx, dw, db = ops.layer_norm_backward(dy, x, mean, rstd)
    assert float(db) == 255 and float(dw) == 3 * 255
    # dx = r (g - g - xh g xh): with one channel and these statistics, -9 dy at the marks and nothing elsewhere
    assert torch.equal(dx[marks, 0], -9 * dy[marks, 0]) and int((dx != 0).sum()) == 8


def test_lost_derivatives_are_errors():
    """Inputs that require a gradient give the 8-bit operators' results bit for bit, and an error where a gradient is asked for; a
    forward-mode tangent is an error everywhere."""
    from torch.autograd import forward_ad
    g = gen(31)
    x, res, w = randn(g, 50, 48), randn(g, 50, 20), randn(g, 48)
    lin = ops.LinearI8.quantize(randn(g, 20, 48))
    xl, rl, wl = (t.clone().requires_grad_(True) for t in (x, res, w))
    q, s = ops.layer_norm_quantize(x, w)
    ql, sl = ops.layer_norm_quantize(xl, wl)
    assert torch.equal(q, ql) and torch.equal(s, sl) and not s.requires_grad
    want, y = ops.matmul_i8(q, s, lin, res=res, out_dtype=F32), ops.matmul_i8(ql, sl, lin, res=rl, out_dtype=F32)
    want2, y2 = ops.linear_i8(x, lin, act="silu"), ops.linear_i8(xl, lin, act="silu")
    assert torch.equal(want, y) and torch.equal(want2, y2)
    for out in (sl, y, y2):
        with pytest.raises(NotImplementedError, match="has no gradient"):
            out.sum().backward()
    with torch.no_grad():
        assert not ops.linear_i8(xl, lin).requires_grad
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, x)
        for call in (lambda: ops.layer_norm(d), lambda: ops.layer_norm(xl, forward_ad.make_dual(w, w)), lambda: ops.linear_i8(d, lin)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        assert torch.equal(ops.layer_norm(x, w), ops.layer_norm(xl, wl).detach())


def test_rows_at_the_end_of_single_precision():
    """Rows whose sums pass the largest number, as documented; the largest rows that do not."""
    x = torch.tensor([[1e38, 1e38, 1e38, 1e38], [1e19, -1e19, 1e19, 3e19], [1e19, -1e19, 8e18, 2e18], [8e37, 8e37, 8e37, 8e37]], device=DEV)
    y, mean, rstd = ops.layer_norm_forward(x, None, torch.full((4,), 0.5, device=DEV))
    assert y[0].isnan().all() and mean[0].isnan()
    assert float(rstd[1]) == 0 and (y[1] == 0.5).all()
    y64, xh, r64 = norm64(x[2:3], None, None, 1e-5)
    within(y[2:3] - 0.5, y64, xh_error(x[2:3], xh, r64) + 4 * U)
    assert (y[3] == 0.5).all()
