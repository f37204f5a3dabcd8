"""The channel-wise operators on NHWC maps -- layer normalisation with its gradient, the product in 8-bit integers, and
the two behind each other -- as measured cases.

A map of N images, H x W pixels and C channels is `rows` = N * H * W rows ("tokens") of C values.  `run` computes a case in
its plain form (elementary torch operations in 32 bits or more) or, where `own` is true, through yolo_amd.ops; `exact` gives
the operators' definition in 64 bits.
"""
import math

import torch

own = False

EPS = 1e-5
_T = {"fp32": torch.float32, "bf16": torch.bfloat16}


# ---- cases ---------------------------------------------------------------------------------------------------------
def _ln(rows, c, x, p, **more):
    """Layer norm over the channels, forward only; x: type of the map, p: type of weight and bias."""
    return dict(more, op="ln", rows=rows, c=c, x=x, p=p)


def _ln_train(rows, c, x, p, **more):
    """Layer norm forward and backward: output, gradient of the map, of weight and of bias."""
    return dict(more, op="ln_train", rows=rows, c=c, x=x, p=p)


def _mm(rows, k, n, y, act, res, **more):
    """Product of rows and weights that both are held in 8 bits, with the epilogue of the framework's convolutions."""
    return dict(more, op="mm", rows=rows, k=k, n=n, y=y, act=act, res=res)


def _lin(rows, k, n, x, act, res, **more):
    """The same from a floating map: its rows are quantised within the call."""
    return dict(more, op="lin", rows=rows, k=k, n=n, x=x, y=x, act=act, res=res)


def _ln_lin(rows, k, n, x, act, **more):
    """Layer norm, quantisation of its rows, product: a pre-norm token-wise layer.  Its output is bf16 for either type of
    map: a value of the norm next to the border between two of the 255 steps falls to either side by the order of a sum."""
    return dict(more, op="ln_lin", rows=rows, k=k, n=n, x=x, p="fp32", y="bf16", act=act, res="none")


def listed():
    return [
        # deepest map of ONE 640-pixel image (20 x 20 x 512): latency of a small call
        _ln(400, 512, "bf16", "bf16", name="ln one image"),
        # stride-8 map of the benchmark's batch, 64 images of 80 x 80 x 128: the largest map a network normalises
        _ln(409600, 128, "bf16", "fp32", name="ln batch 64 stride 8"),
        # training on the stride-16 map of the same batch (40 x 40 x 256)
        _ln_train(102400, 256, "bf16", "fp32", name="ln train batch 64"),
        # single precision, 8 images of 19 x 19, a 255-channel head map: odd rows, nothing aligned
        _ln_train(2888, 255, "fp32", "fp32", name="ln train odd fp32"),
        # one row: a pooled image vector through a 1024 x 1024 layer, or one token: nothing but the weights to read
        _mm(1, 1024, 1024, "bf16", "none", "none", name="mm one row"),
        # 1x1 convolution behind spatial pyramid pooling, 64 images of 19 x 19, 4096 -> 512: the largest product
        _mm(23104, 4096, 512, "bf16", "leaky", "none", name="mm pyramid"),
        # 1x1 convolution of the stride-8 stage, 64 x 80 x 80, 128 -> 128, with a shortcut: bound by the maps
        _mm(409600, 128, 128, "bf16", "silu", "after", name="mm stride 8"),
        # prediction layer on 8 images of 19 x 19: 1000 -> 255, single-precision output, nothing a multiple of the tiles
        _mm(2888, 1000, 255, "fp32", "none", "none", name="mm odd head"),
        # 1x1 convolution of the stride-32 stage of the batch (20 x 20, 512 -> 512) with its shortcut
        _lin(25600, 512, 512, "bf16", "silu", "after", name="linear batch 64"),
        # the same stage for one image, 1024 -> 512: few rows, long sums
        _lin(400, 1024, 512, "bf16", "silu", "none", name="linear one image"),
        # expansion of a token-wise block, 256 -> 1024, on the stride-16 map of the batch
        _ln_lin(102400, 256, 1024, "bf16", "silu", name="ln linear batch 64"),
        # the same block on one small single-precision map (13 x 13)
        _ln_lin(169, 384, 1536, "fp32", "silu", name="ln linear one map"),
    ]


MOST_VALUES, MOST_PRODUCTS = 409600 * 128, 23104 * 4096 * 512


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["ln", "ln_train", "mm", "lin", "ln_lin"])
    t = rng.choice(["bf16", "bf16", "fp32"])
    c = _spread(rng, 16, 4096 if op == "mm" else 2048)
    if rng.random() < 0.5:
        c = (c + 15) // 16 * 16
    rows = _spread(rng, 1, max(1, MOST_VALUES // (2 if t == "fp32" else 1) // c))
    if op in ("ln", "ln_train"):
        return (_ln if op == "ln" else _ln_train)(rows, c, t, rng.choice(["fp32", t]))
    n = _spread(rng, 8, 2048)
    if rng.random() < 0.5:
        n = (n + 15) // 16 * 16
    rows = max(1, min(rows, MOST_VALUES // (2 if t == "fp32" else 1) // n, MOST_PRODUCTS // (c * n)))
    act = rng.choice(["none", "leaky", "silu"])
    if op == "ln_lin":
        return _ln_lin(rows, c, n, t, act)
    return (_mm if op == "mm" else _lin)(rows, c, n, t, act, rng.choice(["none", "after", "before"]))


# ---- inputs --------------------------------------------------------------------------------------------------------
def _map(g, rows, c):
    """A feature map as the networks make them: channels of unlike spread and offset behind a smooth activation."""
    spread = torch.exp(0.5 * torch.randn(c, generator=g, device=g.device))
    x = torch.randn(rows, c, generator=g, device=g.device) * spread + 0.3 * torch.randn(c, generator=g, device=g.device)
    return x * torch.sigmoid(x)


def _to_i8(x):
    """(values in [-127, 127], scales) of rows, for inputs that a program already holds in 8 bits."""
    s = x.abs().amax(1) / 127
    return torch.round(x / s[:, None]).clamp(-127, 127).to(torch.int8), s


def prepare(case, seed):
    dev = "cuda" if torch.cuda.is_available() else "cpu"
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device=dev)
    op, rows = case["op"], case["rows"]
    st = {"case": case}
    width = case["c"] if op in ("ln", "ln_train") else case["k"]
    x = _map(g, rows, width)
    if op in ("ln", "ln_train", "ln_lin"):
        p = _T[case["p"]]
        st["w"], st["b"] = (1 + 0.2 * rnd(width)).to(p), (0.2 * rnd(width)).to(p)
    if op == "mm":
        st["q"], st["qs"] = _to_i8(x)
    else:
        st["x"] = x.to(_T[case["x"]])
    if op == "ln_train":
        st["dy"] = rnd(rows, width).to(_T[case["x"]])
        for k in ("x", "w", "b"):
            st[k].requires_grad_(True)
    if op in ("mm", "lin", "ln_lin"):
        n, y = case["n"], _T[case["y"]]
        st["wq"], st["ws"] = _to_i8(rnd(n, width) / math.sqrt(width))
        st["bias"] = 0.1 * rnd(n)
        st["res"] = rnd(rows, n).to(y) if case["res"] != "none" else None
        st["y"] = y
        if own:   # the weights, laid out once
            from yolo_amd import ops
            st["lin"] = ops.LinearI8(st["wq"], st["ws"], st["bias"])
    return st


# ---- the operators -------------------------------------------------------------------------------------------------
SLOPE = 0.1


def _norm32(x):
    x = x.float()
    x = x - x.mean(1, keepdim=True)
    rstd = torch.rsqrt((x * x).mean(1, keepdim=True) + EPS)
    return x * rstd, rstd


def _quantize32(x):
    # the scale is a / 127 rounded once (a division by a number becomes a product with its reciprocal on the GPU: in 64 bits
    # that ends in the same 32), and the quotient is taken in 64 bits: it is rounded up or down next to a border
    s = (x.abs().amax(1).double() / 127).float()
    return torch.round(x.double() / s.double()[:, None]).float(), s


def _act32(v, act):
    if act == "silu":
        return v * torch.sigmoid(v)
    return torch.where(v > 0, v, v * SLOPE) if act == "leaky" else v


def _product32(q, s, st):
    case, res = st["case"], st["res"]
    v = (q @ st["wq"].float().t()) * s[:, None] * st["ws"] + st["bias"]
    if case["res"] == "before":
        v = v + res.float()
    v = _act32(v, case["act"])
    if case["res"] == "after":
        v = v + res.float()
    return v.to(st["y"])


@torch.no_grad()
def _plain(st):
    case = st["case"]
    op = case["op"]
    if op in ("ln", "ln_train", "ln_lin"):
        x, w = st["x"], st["w"].float()
        xh, rstd = _norm32(x)
        y = xh * w + st["b"].float()
        if op == "ln":
            return y.to(x.dtype)
        if op == "ln_lin":
            return _product32(*_quantize32(y), st)
        dy = st["dy"].float()
        gw = dy * w
        dx = rstd * (gw - gw.mean(1, keepdim=True) - xh * (gw * xh).mean(1, keepdim=True))
        return y.to(x.dtype), dx.to(x.dtype), (dy * xh).sum(0).to(st["w"].dtype), dy.sum(0).to(st["b"].dtype)
    if op == "lin":
        return _product32(*_quantize32(st["x"]), st)
    return _product32(st["q"].float(), st["qs"], st)


def run(st):
    if not own:
        return _plain(st)
    from yolo_amd import ops
    case = st["case"]
    op = case["op"]
    if op == "ln":
        return ops.layer_norm(st["x"], st["w"], st["b"], EPS)
    if op == "ln_train":
        y = ops.layer_norm(st["x"], st["w"], st["b"], EPS)
        return (y.detach(),) + torch.autograd.grad(y, (st["x"], st["w"], st["b"]), st["dy"])
    how = dict(act=case["act"], slope=SLOPE, res=st["res"], res_mode="after" if case["res"] == "none" else case["res"],
               out_dtype=st["y"])
    if op == "mm":
        return ops.matmul_i8(st["q"], st["qs"], st["lin"], **how)
    if op == "lin":
        return ops.linear_i8(st["x"], st["lin"], **how)
    q, s = ops.layer_norm_quantize(st["x"], st["w"], st["b"], EPS)
    return ops.matmul_i8(q, s, st["lin"], **how)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    size = {"bf16": 2, "fp32": 4}
    op, rows = case["op"], case["rows"]
    if op == "ln":
        c = case["c"]
        return {"bytes": 2 * rows * c * size[case["x"]] + 2 * c * size[case["p"]], "flops": 8 * rows * c}
    if op == "ln_train":      # the map, its output, the output's gradient and the map's; weight, bias and their gradients
        c = case["c"]
        return {"bytes": 4 * rows * c * size[case["x"]] + 4 * c * size[case["p"]], "flops": 22 * rows * c}
    k, n = case["k"], case["n"]
    y = size[case["y"]]
    read = rows * k + 4 * rows if op == "mm" else rows * k * size[case["x"]]
    if op == "ln_lin":
        read += 2 * k * size[case["p"]]
    maps = 2 if case["res"] != "none" else 1
    return {"bytes": read + n * k + 8 * n + maps * rows * n * y, "flops": 2 * rows * n * k}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------
@torch.no_grad()
def exact(case, seed):
    st = prepare({k: v for k, v in case.items()}, seed)
    d = {k: v.detach().double() for k, v in st.items() if isinstance(v, torch.Tensor)}
    op = case["op"]
    if op in ("ln", "ln_train", "ln_lin"):
        x, c = d["x"], d["x"].shape[1]
        mean = x.sum(1) / c
        var = (x - mean[:, None]).pow(2).sum(1) / c
        sigma = (var + EPS).sqrt()
        unit = (x - mean[:, None]) / sigma[:, None]
        out = unit * d["w"] + d["b"]
        if op == "ln":
            return out
        if op == "ln_train":
            dy = d["dy"]
            # dx_j = sum_i dy_i w_i d(unit_i)/dx_j, d(unit_i)/dx_j = (delta_ij - 1/c - unit_i unit_j / c) / sigma
            t = dy * d["w"]
            dx = (t - t.sum(1)[:, None] / c - unit * ((t * unit).sum(1)[:, None] / c)) / sigma[:, None]
            return out, dx, torch.einsum("rc,rc->c", dy, unit), dy.sum(0)
        q_in = out
    else:
        q_in = d.get("x")
    if op == "mm":
        q, s = d["q"], d["qs"]
    else:
        top = q_in.abs().max(1).values
        s = (top / 127).float().double()      # a scale is held in single precision
        q = torch.round(q_in / s[:, None])
    acc = torch.mm(q, d["wq"].t().contiguous())
    v = acc * torch.outer(s, d["ws"]) + d["bias"]
    if case["res"] == "before":
        v = v + d["res"]
    if case["act"] == "silu":
        v = v / (1 + torch.exp(-v))
    elif case["act"] == "leaky":
        v = torch.maximum(v, 0 * v) + SLOPE * torch.minimum(v, 0 * v)
    if case["res"] == "after":
        v = v + d["res"]
    return v
