"""CPU-side checks of the layer-norm and 8-bit entry points: struct layouts, workspace sizes, and that every bad argument is
turned away before anything is launched (addresses here are numbers that nothing reads)."""
import ctypes as C
import os
import subprocess

import pytest
import torch

from helpers import ROOT
from yolo_amd import _ffi, ops

P = 1 << 20        # an aligned address


def test_struct_layouts():
    names = ("ydet_layer_norm_desc", "ydet_layer_norm_grad_desc", "ydet_quantize_desc", "ydet_matmul_i8_desc")
    last = ("eps", "param_dtype", "eps", "out_dtype")
    src = '#include <stddef.h>\n#include <stdio.h>\n#include "ydet.h"\nint main(){' + "".join(
        f'printf("%zu %zu ", sizeof({n}), offsetof({n}, {f}));' for n, f in zip(names, last)) + "return 0;}"
    exe = os.path.join(ROOT, "build", "abi_rows")
    os.makedirs(os.path.dirname(exe), exist_ok=True)
    subprocess.run(["gcc", "-x", "c", "-", "-I", os.path.join(ROOT, "include"), "-o", exe], input=src.encode(), check=True)
    got = [int(v) for v in subprocess.run([exe], capture_output=True, check=True).stdout.split()]
    mine = (_ffi.LayerNormDesc, _ffi.LayerNormGradDesc, _ffi.QuantizeDesc, _ffi.MatmulI8Desc)
    assert got == [v for m, f in zip(mine, last) for v in (C.sizeof(m), getattr(m, f).offset)]


def ln(**kw):
    d = dict(x=P, y=P, gamma=P, beta=P, mean=None, rstd=None, rows=4, C=32, x_ld=32, x_coff=0, y_ld=32, y_coff=0, dtype=0, param_dtype=0,
             eps=1e-5)
    d.update(kw)
    return _ffi.lib().ydet_layer_norm(_ffi.LayerNormDesc(**d), None)


def grad(ws=P, ws_bytes=1 << 30, **kw):
    d = dict(dy=P, x=P, dx=P, gamma=P, mean=P, rstd=P, dgamma=P, dbeta=P, rows=4, C=32, dy_ld=32, dy_coff=0, x_ld=32, x_coff=0, dx_ld=32,
             dx_coff=0, dtype=0, param_dtype=0)
    d.update(kw)
    return _ffi.lib().ydet_layer_norm_backward(_ffi.LayerNormGradDesc(**d), ws, ws_bytes, None)


def quant(**kw):
    d = dict(x=P, q=P, scale=P, gamma=None, beta=None, rows=4, C=20, x_ld=20, x_coff=0, q_ld=32, dtype=0, param_dtype=0, normalize=0, eps=0.0)
    d.update(kw)
    return _ffi.lib().ydet_quantize_rows_i8(_ffi.QuantizeDesc(**d), None)


def product(**kw):
    d = dict(x=P, x_scale=P, w=P, w_scale=P, bias=P, res=None, y=P, rows=4, K=64, N=32, kp=64, n_pad=128, x_ld=64, x_coff=0, y_ld=32,
             y_coff=0, res_ld=0, res_coff=0, act=0, slope=0.0, res_mode=0, out_dtype=1)
    d.update(kw)
    return _ffi.lib().ydet_matmul_i8(_ffi.MatmulI8Desc(**d), None, 0, None)


def linear(ws=P, ws_bytes=1 << 40, rows=4, C_=64, **kw):
    q = _ffi.QuantizeDesc(x=P, rows=rows, C=C_, x_ld=C_, dtype=1, param_dtype=0)
    d = dict(w=P, w_scale=P, bias=P, y=P, rows=4, K=64, N=32, kp=64, n_pad=128, y_ld=32, out_dtype=1)
    d.update(kw)
    return _ffi.lib().ydet_linear_i8(q, _ffi.MatmulI8Desc(**d), ws, ws_bytes, None)


ARG, WS = -1, -3


@pytest.mark.parametrize("call,kw,text", [
    (ln, dict(x=None), "null"), (ln, dict(y=None), "null"), (ln, dict(rows=-1), "rows"), (ln, dict(rows=1 << 31), "rows"), (ln, dict(C=0), "C="),
    (ln, dict(C=8193, x_ld=9000, y_ld=9000), "C="), (ln, dict(x_ld=31), "slice"), (ln, dict(y_coff=1), "slice"), (ln, dict(x_coff=-1), "slice"),
    (ln, dict(dtype=2), "dtype"), (ln, dict(param_dtype=7), "dtype"), (ln, dict(eps=-1.0), "eps"), (ln, dict(eps=float("nan")), "eps"),
    (ln, dict(mean=P), "together"), (ln, dict(x=P + 2), "misaligned"),
    (grad, dict(x=None), "null"), (grad, dict(mean=None), "null"), (grad, dict(rows=-5), "rows"), (grad, dict(C=8193), "C="),
    (grad, dict(dx_ld=16), "slice"), (grad, dict(dy_coff=3), "slice"), (grad, dict(dtype=5), "dtype"), (grad, dict(ws=None), "workspace"),
    (grad, dict(dgamma=P + 1), "misaligned"),
    (quant, dict(x=None), "null"), (quant, dict(scale=None), "null"), (quant, dict(q_ld=20), "q_ld"), (quant, dict(q_ld=16), "q_ld"),
    (quant, dict(q=P + 8), "misaligned"), (quant, dict(C=21), "slice"), (quant, dict(normalize=1, eps=-1.0), "eps"), (quant, dict(rows=-1), "rows"),
    (product, dict(x=None), "null"), (product, dict(x_scale=None), "null"), (product, dict(w=None), "null"), (product, dict(y=None), "null"),
    (product, dict(res_mode=1, res_ld=32), "null"), (product, dict(res_mode=1, res=P, res_ld=31), "residual"), (product, dict(K=0), "K="),
    (product, dict(K=131072, kp=131072, x_ld=131072), "K="), (product, dict(kp=96), "padded"), (product, dict(K=65, x_ld=80), "padded"),
    (product, dict(n_pad=64), "padded"), (product, dict(N=129, y_ld=160), "padded"), (product, dict(x_ld=63), "slice"), (product, dict(y_coff=1), "slice"),
    (product, dict(x_ld=(1 << 23) + 16), "x_ld"), (product, dict(out_dtype=2), "out_dtype"), (product, dict(act=3), "act"), (product, dict(res_mode=3), "act"),
    (product, dict(w=P + 8), "alignment"), (product, dict(w_scale=P + 4), "alignment"), (product, dict(y=P + 1), "misaligned"),
    (product, dict(rows=(1 << 31) - 1), "rows"),
    (linear, dict(rows=5), "product of"), (linear, dict(C_=65), "product of"), (linear, dict(w=None), "null"), (linear, dict(N=200, y_ld=200), "padded"),
    (linear, dict(rows=1 << 20, C_=8193, K=8193, kp=8256), "product of"), (linear, dict(C_=8193, K=8193, kp=8256), "K="),
    (linear, dict(rows=1 << 16, ws=None, **{"N": 32}), "product of")])
def test_bad_arguments(call, kw, text):
    assert call(**kw) == ARG
    assert text in _ffi.lib().ydet_last_error().decode()


def test_workspace():
    size = _ffi.lib().ydet_layer_norm_backward_workspace_bytes
    assert size(-1, 32) == size(4, 0) == size(4, 8193) == 0
    assert size(0, 32) == size(1, 32) == 2 * 32 * 4
    for C_ in (1, 255, 2048, 8192):
        sizes = [size(r, C_) for r in (1, 100, 10000, 1 << 20, (1 << 31) - 1)]
        assert sizes == sorted(sizes) and sizes[-1] <= 1024 * 2 * C_ * 4
    assert grad(ws_bytes=size(4, 32) - 4) == WS
    assert "workspace" in _ffi.lib().ydet_last_error().decode()


def test_linear_workspace():
    lib = _ffi.lib()

    def sizes(rows, K, N, **kw):
        q = _ffi.QuantizeDesc(x=P, rows=rows, C=K, x_ld=K, dtype=1, **kw)
        kp, n_pad = (K + 63) // 64 * 64, (N + 127) // 128 * 128
        d = _ffi.MatmulI8Desc(w=P, w_scale=P, y=P, rows=rows, K=K, N=N, kp=kp, n_pad=n_pad, y_ld=N, out_dtype=1)
        return q, d, lib.ydet_linear_i8_workspace_bytes(q, d)
    assert sizes(1, 1024, 1024)[2] == 0 and sizes(100, 2048, 512)[2] == 0           # one launch
    assert sizes(100, 2049, 512)[2] == 100 * 2064 + 100 * 4 and sizes(400, 1024, 512)[2] == 400 * 1028 and sizes(25601, 500, 64)[2] == 25601 * 512 + 25604 * 4
    q, d, n = sizes(25600, 500, 64)
    assert lib.ydet_linear_i8(q, d, P, n - 1, None) == WS and "workspace" in lib.ydet_last_error().decode()
    assert lib.ydet_linear_i8(q, d, None, n, None) == ARG
    assert lib.ydet_linear_i8(q, d, P + 8, n, None) == ARG
    assert sizes(4, 8193, 8)[2] == 0 and sizes(0, 64, 64)[2] == 0
    # rows of x at odd addresses need a copy where they are many
    rows = lambda n, ld: _ffi.MatmulI8Desc(x=P, x_scale=P, w=P, w_scale=P, y=P, rows=n, K=77, N=64, kp=128, n_pad=128, x_ld=ld, y_ld=64, out_dtype=1)
    size = lib.ydet_matmul_i8_workspace_bytes
    assert size(rows(100, 77)) == 0 and size(rows(50000, 80)) == 0 and size(rows(50000, 77)) == 50000 * 80 and size(rows(-1, 77)) == 0
    assert lib.ydet_matmul_i8(rows(50000, 77), None, 0, None) == WS and lib.ydet_matmul_i8(rows(50000, 77), P + 4, 1 << 30, None) == ARG


def test_nothing_to_do_is_no_error():
    assert ln(rows=0, x=None, y=None) == 0
    assert quant(rows=0, x=None, q=None, scale=None) == 0
    assert product(rows=0, x=None, y=None) == 0
    assert grad(dx=None, dgamma=None, dbeta=None, ws=None, ws_bytes=0) == 0
    assert grad(rows=0, dgamma=None, dbeta=None, ws=None, ws_bytes=0) == 0


def test_cpu_tensors_are_refused():
    x = torch.randn(3, 16)
    for call in (lambda: ops.layer_norm(x), lambda: ops.layer_norm(x.requires_grad_(True)), lambda: ops.layer_norm_forward(x),
                 lambda: ops.quantize_rows(x), lambda: ops.layer_norm_quantize(x), lambda: ops.LinearI8.quantize(x),
                 lambda: ops.LinearI8(torch.zeros(2, 4, dtype=torch.int8), torch.ones(2))):
        with pytest.raises(RuntimeError):
            call()


# ---- the planner's choice of 8-bit layers ---------------------------------------------------------------------------------------
def test_which_layers_go_to_8_bits():
    from yolo_amd import engine
    assert engine._pointwise_int8 is False
    pays = engine.pointwise_int8_pays
    assert pays(361, 4096, 512) and pays(400, 512, 512) and pays(6400, 2048, 1024) and pays(25600, 512, 2048) and pays(102400, 256, 1024)
    assert not pays(25600, 512, 512) and not pays(102400, 1024, 256) and not pays(409600, 128, 512) and not pays(400, 256, 256)
    g = engine.Graph("cpu", "bf16")
    x = g.input_nchw(1, 512, 20, 20)
    conv = lambda i, o, k=1, s=1, **kw: torch.nn.Conv2d(i, o, k, s, k // 2, **kw)
    g.conv(x, conv(512, 512))                                   # 1: taken
    g.conv(x, conv(512, 512, 3))                                # not 1x1
    g.conv(x, conv(512, 512, 1, 2))                             # strided
    g.conv(x, conv(512, 512, groups=2))                         # grouped
    g.conv(x, conv(512, 255))                                   # prediction layer: no whole pieces
    g.conv(x, conv(512, 512), out_dtype=_ffi.F32)               # fp32 map
    y = g.conv(x, conv(512, 64))                                # 7: taken
    g.conv(y, conv(64, 64))                                     # short sums
    g.conv(x, conv(512, 512), post=(torch.nn.BatchNorm2d(512), None, _ffi.ACT_LEAKY, 0.1))      # a second stage
    g.conv(x, conv(512, 512), res=x, res_mode=_ffi.RES_AFTER_ACT)                               # 10: taken
    assert g.pointwise_int8() == [1, 7, 10]
    engine.set_pointwise_int8(True)
    try:
        plan = g.finalize()                                     # (no GPU here: nothing is replaced)
    finally:
        engine.set_pointwise_int8(False)
    assert not any(k == "linear_i8" for k, _ in plan.g.ops) and plan.i8_ws == [None]


# ---- batches without rows: nothing is launched, so the wrappers run here up to the library's own return -----------------------
@pytest.fixture
def without_gpu(monkeypatch):
    monkeypatch.setattr(ops, "_need_cuda", lambda *t: None)
    monkeypatch.setattr(ops, "_launch", lambda dev, call, *args: call(*args, None))


@pytest.mark.parametrize("lead", [(0,), (3, 0), (0, 5)])
@pytest.mark.parametrize("K", [30, 32, 64, 77, 1024])
def test_products_without_rows(without_gpu, K, lead):
    """Whatever the rows' pitch (a multiple of 4 or not): an empty output of the right shape."""
    lin = ops.LinearI8(torch.ones(20, K, dtype=torch.int8), torch.ones(20), torch.ones(20))
    x = torch.empty(*lead, K)
    q, s = ops.quantize_rows(x)
    assert q.shape == lead + (K,) and s.shape == lead
    for rows in (q, torch.empty(*lead, K, dtype=torch.int8)):
        y = ops.matmul_i8(rows, s, lin, act="silu")
        assert y.shape == lead + (20,) and y.dtype == torch.bfloat16
        assert ops.matmul_i8(rows, s, lin, res=torch.empty(*lead, 20), out_dtype=torch.float32).shape == lead + (20,)
    assert ops.matmul_i8(*ops.layer_norm_quantize(x), lin).shape == lead + (20,)
    assert ops.linear_i8(x, lin).shape == lead + (20,)


def test_few_rows_in_place_need_a_workspace():
    """An output over the floating rows never takes the one launch; beside them, also in the same rows, it does.  (A workspace that is
    too small or misaligned says that two launches would be taken, a bad type of the rows that the one launch was reached: nothing is
    launched here.)"""
    lib = _ffi.lib()

    def meets(rows=16, K=64, N=64, x=P, y=P, x_ld=64, y_ld=64, x_coff=0, y_coff=0, dtype=1, out=1):
        q = _ffi.QuantizeDesc(x=x, rows=rows, C=K, x_ld=x_ld, x_coff=x_coff, dtype=dtype, param_dtype=7)
        d = _ffi.MatmulI8Desc(w=P, w_scale=P, y=y, rows=rows, K=K, N=N, kp=(K + 63) // 64 * 64, n_pad=(N + 127) // 128 * 128, y_ld=y_ld,
                              y_coff=y_coff, out_dtype=out)
        bytes_ = rows * ((K + 15) // 16 * 16) + (rows + 3) // 4 * 16
        rc = lib.ydet_linear_i8(q, d, P, bytes_ - 1, None)
        text = lib.ydet_last_error().decode()
        assert (rc == WS and f"{bytes_ - 1} < {bytes_}" in text) or (rc == ARG and "dtype" in text)
        assert lib.ydet_linear_i8(q, d, None, 0, None) in (ARG, WS)
        return rc == WS
    assert meets()                                                          # in place
    assert not meets(y=P + 16 * 128) and not meets(y=P - 16 * 128)          # behind and before
    assert meets(y=P + 16 * 128 - 2) and meets(y=P - 16 * 128 + 2)          # over the last and the first value
    for x0, y0, m in ((0, 64, False), (64, 0, False), (0, 63, True), (63, 0, True), (0, 0, True), (1, 65, False), (65, 1, False)):
        assert meets(x_ld=129, y_ld=129, x_coff=x0, y_coff=y0) == m, (x0, y0)
    wide = dict(x_ld=200, y_ld=200)
    assert not meets(**wide, y=P + 3 * 400, y_coff=100)                     # other rows, other columns
    assert not meets(**wide, y=P + 3 * 400, y_coff=180, N=20)
    assert meets(**wide, x=P + 2 * 100, N=120)                              # (columns 0 .. 119 and 100 .. 163)
    assert not meets(**wide, y=P + 2 * 180, N=20) and meets(**wide, y=P + 2 * 180, N=21)      # up to the next row of x, into it
    assert meets(x_ld=128, y_ld=256, y_coff=64)                             # other pitches: their ranges meet
    # other types of rows and output
    assert not meets(dtype=0, out=1, x_ld=128, y_ld=256, y_coff=128) and meets(dtype=0, out=1, x_ld=128, y_ld=256, y_coff=127)
    assert not meets(rows=1, y=P + 128) and meets(rows=1, y=P + 126)


# ---- derivatives that the operators do not have are errors, not constants (the library's calls are left out: values do not matter) --
@pytest.fixture
def no_launches(monkeypatch):
    monkeypatch.setattr(ops, "_need_cuda", lambda *t: None)
    monkeypatch.setattr(ops, "_launch", lambda dev, call, *args: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)


def _operators():
    """name -> (call of a floating [4, 32] tensor in every place that takes one, whether it has a gradient)"""
    lin = ops.LinearI8(torch.ones(8, 32, dtype=torch.int8), torch.ones(8))
    q, s, x = torch.ones(4, 32, dtype=torch.int8), torch.ones(4), torch.ones(4, 32)
    F = torch.float32
    return {"layer_norm": lambda t: ops.layer_norm(t), "layer_norm weight": lambda t: ops.layer_norm(x, t[0]),
            "layer_norm bias": lambda t: ops.layer_norm(x, None, t[0]), "layer_norm_forward": lambda t: ops.layer_norm_forward(t)[0],
            "layer_norm_backward dy": lambda t: ops.layer_norm_backward(t, x, s, s)[0],
            "layer_norm_backward rstd": lambda t: ops.layer_norm_backward(x, x, s, t[:, 0])[0],
            "quantize_rows": lambda t: ops.quantize_rows(t)[1], "layer_norm_quantize": lambda t: ops.layer_norm_quantize(t)[1],
            "layer_norm_quantize weight": lambda t: ops.layer_norm_quantize(x, t[0])[1],
            "matmul_i8 scale": lambda t: ops.matmul_i8(q, t[:, 0], lin, out_dtype=F), "matmul_i8 res": lambda t: ops.matmul_i8(q, s, lin, res=t[:, :8], out_dtype=F),
            "linear_i8": lambda t: ops.linear_i8(t, lin), "linear_i8 res": lambda t: ops.linear_i8(x, lin, res=t[:, :8])}


NAMES = ["layer_norm", "layer_norm weight", "layer_norm bias", "layer_norm_forward", "layer_norm_backward dy", "layer_norm_backward rstd",
         "quantize_rows", "layer_norm_quantize", "layer_norm_quantize weight", "matmul_i8 scale", "matmul_i8 res", "linear_i8", "linear_i8 res"]


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused(no_launches, name):
    from torch.autograd import forward_ad as fwd
    call = _operators()[name]
    x = torch.ones(4, 32)
    with fwd.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(fwd.make_dual(x, x))
        call(x)                                         # (nothing dual: as ever)
        with torch.no_grad():
            call(x)
    call(x)
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.jvp(call, (x,), (x,))


def test_no_dimension_is_refused(no_launches):
    for grad in (False, True):
        with pytest.raises(ValueError, match="at least one channel"):
            ops.layer_norm(torch.tensor(1.0, requires_grad=grad))


def test_forward_mode_through_the_backward_pass_is_refused(no_launches):
    from torch.autograd import forward_ad as fwd
    x = torch.ones(4, 32, requires_grad=True)
    with fwd.dual_level():
        y = ops.layer_norm(x)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(y, x, fwd.make_dual(torch.ones(4, 32), torch.ones(4, 32)))


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning", "ignore::DeprecationWarning")
@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name", NAMES)
def test_tracing_is_refused(no_launches, name, grad):
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(_operators()[name], torch.ones(4, 32, requires_grad=grad), check_trace=False)


@pytest.mark.parametrize("name", [n for n in NAMES if n.split()[0] in ("quantize_rows", "layer_norm_quantize", "matmul_i8", "linear_i8")])
def test_gradients_of_8_bit_operators_are_errors(no_launches, name):
    call = _operators()[name]
    x = torch.ones(4, 32)
    assert not call(x).requires_grad
    leaf = x.clone().requires_grad_(True)
    with torch.no_grad():
        assert not call(leaf).requires_grad
    assert not call(leaf.detach()).requires_grad
    y = call(leaf)                                      # the call itself is as before
    with pytest.raises(NotImplementedError, match=f"{'quantize_rows' if 'quantize' in name else name.split()[0]} has no gradient"):
        (y.sum() + leaf.sum()).backward()
    assert leaf.grad is None


@pytest.mark.parametrize("shape", [(4,), (2, 2)])
def test_results_of_8_bit_operators_may_be_changed_in_place(no_launches, shape):
    """As before there was an error to record, also where the result is laid out in more than two dimensions."""
    lin = ops.LinearI8(torch.ones(8, 32, dtype=torch.int8), torch.ones(8))
    x = torch.ones(*shape, 32, requires_grad=True)
    for y in (ops.linear_i8(x, lin), ops.quantize_rows(x)[1], ops.matmul_i8(torch.ones(*shape, 32, dtype=torch.int8), *ops.quantize_rows(x)[1:], lin)):
        y.zero_()
        y += 1
        y[..., :1].mul_(2)
        assert y.shape[:len(shape)] == shape and float(y.detach().flatten()[0]) == 2
        with pytest.raises(NotImplementedError, match="has no gradient"):
            y.sum().backward()


def test_no_gradient_through_a_block_of_8_bit_operators(no_launches):
    lin = ops.LinearI8(torch.ones(8, 32, dtype=torch.int8), torch.ones(8))
    w = torch.ones(32, requires_grad=True)
    y = ops.matmul_i8(*ops.layer_norm_quantize(torch.ones(4, 32), w), lin, out_dtype=torch.float32)
    with pytest.raises(NotImplementedError, match="has no gradient"):
        y.sum().backward()
    # a weight of another type than the bias, which is converted on the way
    s = ops.layer_norm_quantize(torch.ones(4, 32), torch.ones(32, dtype=torch.bfloat16, requires_grad=True), torch.ones(32))[1]
    with pytest.raises(NotImplementedError, match="has no gradient"):
        s.sum().backward()


def test_8_bits_are_chosen_where_they_were_measured_to_pay():
    """Both sides of every border of the rule, with the measured times (us, bf16 kernel / 8 bits)."""
    from yolo_amd.engine import pointwise_int8_pays as pays
    better = [(49, 512, 64, 8, 6), (2704, 512, 512, 9.6, 8.7), (1600, 768, 2048, 14, 12), (3249, 1024, 512, 15, 12), (6400, 2048, 512, 26, 24),
              (6400, 4096, 64, 42, 30), (6656, 1024, 2048, 37, 34), (16384, 1024, 4096, 152, 126), (25600, 512, 1024, 42, 39), (102400, 512, 1024, 161, 135),
              (46208, 256, 1024, 55, 46), (92416, 384, 1536, 190, 148), (49, 256, 512, 7, 5), (169, 384, 768, 8, 7)]
    worse = [(5776, 512, 1024, 14, 16), (6400, 512, 64, 9, 10), (6400, 768, 1024, 17, 22), (6400, 1024, 512, 16, 18),
             (6656, 512, 1024, 15, 18), (16384, 512, 1024, 25, 29), (204800, 512, 1024, 301, 325), (409600, 256, 512, 195, 273), (204800, 256, 1024, 192, 212),
             (25600, 256, 1024, 29, 30), (102400, 256, 512, 57, 60), (3249, 256, 512, 7, 8), (6656, 256, 1024, 10, 13), (102400, 1024, 256, 81, 115)]
    assert all(pays(*r[:3]) for r in better)
    assert not any(pays(*r[:3]) for r in worse)
    assert all(b > i for *_, b, i in better) and all(b < i for *_, b, i in worse)
