"""Tensor-level wrappers of the decode / NMS / IoU, layer-norm and 8-bit entry points of libydet.so.

Inputs and outputs are CUDA tensors; everything is enqueued on torch's current stream and nothing
here synchronises with the host.
"""
import ctypes as C

import torch
from torch.autograd import forward_ad

from . import _ffi


def _dt(t):
    if t.dtype == torch.float32:
        return _ffi.F32
    if t.dtype == torch.bfloat16:
        return _ffi.BF16
    raise TypeError(f"unsupported dtype {t.dtype}")


def _need_cuda(*ts):
    for t in ts:
        if not t.is_cuda:
            raise RuntimeError("yolo_amd GPU operator called with a CPU tensor (there is no CPU path here)")


def decode_v5(heads, strides, anchors_px, na, no, grid_transposed=False, row_max=True):
    """heads: NHWC maps [N, ny, nx, >=na*no] (fp32 or bf16, last dim contiguous), one per level.
    strides: per-level float; anchors_px: per-level list of 2*na pixel sizes.
    Returns z [N, sum(na*ny*nx), no] fp32 (yolov5_official/model.py:56-81).
    With row_max, the kernel also emits per box max_c(cls_c * obj); it rides on the result as `z._ydet_row_max`
    (tensor, version of z) and lets nms_v5 skip its scan of z while z stays unmodified."""
    _need_cuda(*heads)
    lib = _ffi.lib()
    nl = len(heads)
    N = heads[0].shape[0]
    levels = (_ffi.V5Level * nl)()
    rows = 0
    for l, h in enumerate(heads):
        assert h.dim() == 4 and h.stride(3) == 1 and h.shape[0] == N
        assert h.stride(2) == h.stride(1) // h.shape[2] and h.stride(0) == h.stride(1) * h.shape[1], "head not NHWC-dense"
        L = levels[l]
        L.head, L.ny, L.nx, L.ld = h.data_ptr(), h.shape[1], h.shape[2], h.stride(2)
        L.stride = float(strides[l])
        for i, v in enumerate(anchors_px[l]):
            L.anchor_wh[i] = float(v)
        rows += na * h.shape[1] * h.shape[2]
    out = torch.empty(N, rows, no, device=heads[0].device, dtype=torch.float32)
    rm = torch.empty(N, rows, device=out.device, dtype=torch.float32) if row_max and no > 5 else None
    with torch.cuda.device(out.device):
        _ffi.check(lib.ydet_decode_v5(levels, nl, N, na, no, int(grid_transposed), _dt(heads[0]), out.data_ptr(),
                                      rm.data_ptr() if rm is not None else None, _ffi.current_stream()),
                   "ydet_decode_v5")
    if rm is not None:
        out._ydet_row_max = (rm, out._version)
    return out


def row_max_of(pred):
    """The row maxima decode_v5 attached to `pred`, if `pred` is still that very tensor, unmodified."""
    hint = getattr(pred, "_ydet_row_max", None)
    if hint is None:
        return None
    rm, version = hint
    if version != pred._version or rm.shape != pred.shape[:2] or rm.device != pred.device:
        return None
    return rm


def decode_v2v3(heads, anchors, A, nc, mode, input_size, mult=32.0, grid_transposed=True):
    """heads: NHWC maps [N, H, W, >=A*(5+nc)] fine -> coarse; anchors: per-level list of 2*A values.
    mode 0 = utils/utils.py xywh_to_xxyy ("v2"), 1 = xywh_to_xxyyv3.
    Returns (boxes [N, n, 4] normalised+clamped xyxy, scores [N, n, nc]) fp32."""
    _need_cuda(*heads)
    lib = _ffi.lib()
    nl = len(heads)
    N = heads[0].shape[0]
    levels = (_ffi.FALevel * nl)()
    n = 0
    for l, h in enumerate(heads):
        assert h.dim() == 4 and h.stride(3) == 1 and h.shape[0] == N
        assert h.stride(2) == h.stride(1) // h.shape[2] and h.stride(0) == h.stride(1) * h.shape[1], "head not NHWC-dense"
        L = levels[l]
        L.head, L.H, L.W, L.ld = h.data_ptr(), h.shape[1], h.shape[2], h.stride(2)
        for i, v in enumerate(anchors[l]):
            L.anchor_wh[i] = float(v)
        n += A * h.shape[1] * h.shape[2]
    dev = heads[0].device
    boxes = torch.empty(N, n, 4, device=dev, dtype=torch.float32)
    scores = torch.empty(N, n, nc, device=dev, dtype=torch.float32)
    with torch.cuda.device(dev):
        _ffi.check(lib.ydet_decode_v2v3(levels, nl, N, A, nc, int(mode), float(mult), float(input_size),
                                        int(grid_transposed), _dt(heads[0]), boxes.data_ptr(), scores.data_ptr(),
                                        _ffi.current_stream()), "ydet_decode_v2v3")
    return boxes, scores


def nms_v5(pred, conf_thres=0.25, iou_thres=0.45, multi_label=False, agnostic=False, max_det=300, max_nms=None,
           max_wh=4096.0, classes=None, row_max="auto"):
    """pred [N, nboxes, 5+nc] fp32 CUDA.  Returns (det [N, max_det, 6], count [N] int32) on the device;
    det rows are (x1, y1, x2, y2, score, cls) in descending score order.
    row_max: "auto" uses the row maxima decode_v5 attached to `pred` (if still valid), None forces the scan."""
    _need_cuda(pred)
    lib = _ffi.lib()
    rm = row_max_of(pred) if isinstance(row_max, str) else row_max
    if pred.dtype != torch.float32 or not pred.is_contiguous():
        rm = None
    if pred.dtype != torch.float32:
        pred = pred.float()
    pred = pred.contiguous()
    N, nboxes, no = pred.shape
    max_nms = max_det if max_nms is None else max_nms
    dev = pred.device
    det = torch.empty(N, max_det, 6, device=dev, dtype=torch.float32)
    count = torch.empty(N, device=dev, dtype=torch.int32)
    if N == 0 or nboxes == 0:
        return det.zero_(), count.zero_()
    ws_bytes = lib.ydet_nms_v5_workspace_bytes(N, nboxes, no)
    ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
    mask_ptr = None
    if classes is not None:
        m = torch.zeros(no - 5, dtype=torch.uint8)
        m[torch.as_tensor(list(classes), dtype=torch.long)] = 1
        mask = m.to(dev)
        mask_ptr = mask.data_ptr()
    with torch.cuda.device(dev):
        _ffi.check(lib.ydet_nms_v5(pred.data_ptr(), N, nboxes, no, float(conf_thres), float(iou_thres),
                                   int(bool(multi_label)), int(bool(agnostic)), int(max_nms), int(max_det),
                                   float(max_wh), mask_ptr, rm.data_ptr() if rm is not None else None,
                                   det.data_ptr(), count.data_ptr(), ws.data_ptr(), ws_bytes,
                                   _ffi.current_stream()), "ydet_nms_v5")
    return det, count


NMS2_METHODS = {"hard_nms_batch": 0, "hard_nms": 1, "hard_nms_myself": 2, "and": 3, "merge": 4, "soft_nms": 5, "diou_nms": 6}


def nms2(pred, conf_thres=0.25, nms_thres=0.6, multi_cls=True, method="diou_nms"):
    """pred [N, nboxes, 5+nc] fp32 CUDA -> (rows [N, cap, 6], count [N] int32, overflow [1] int32) on the device:
    yolov5_official/utils.py:318-460, rows (x1, y1, x2, y2, score, cls) in descending score order."""
    _need_cuda(pred)
    if method not in NMS2_METHODS:
        raise ValueError(f"unknown NMS method {method!r}")
    if method == "merge" and not nms_thres < 1.0:
        raise ValueError("merge needs nms_thres < 1 (the reference does not terminate otherwise)")
    lib = _ffi.lib()
    pred = pred.float().contiguous()
    N, nboxes, no = pred.shape
    dev = pred.device
    m = NMS2_METHODS[method]
    cap = min(lib.ydet_nms2_out_cap(no, m), max(nboxes * (no - 5), 1))
    rows = torch.empty(N, cap, 6, device=dev, dtype=torch.float32)
    count = torch.zeros(N, device=dev, dtype=torch.int32)
    overflow = torch.zeros(1, device=dev, dtype=torch.int32)
    if N == 0 or nboxes == 0:
        return rows, count, overflow
    ws_bytes = lib.ydet_nms2_workspace_bytes(N, nboxes, no, m)
    ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
    with torch.cuda.device(dev):
        _ffi.check(lib.ydet_nms2(pred.data_ptr(), N, nboxes, no, float(conf_thres), float(nms_thres), int(bool(multi_cls)), m,
                                 rows.data_ptr(), cap, count.data_ptr(), overflow.data_ptr(), ws.data_ptr(), ws_bytes,
                                 _ffi.current_stream()), "ydet_nms2")
    return rows, count, overflow


def nms_cluster_diou(pred, conf_thres=0.1, iou_thres=0.6, max_box=1500, classes=None, agnostic=False):
    """pred [N, nboxes, 5+nc] fp32 CUDA -> (rows [N, max_box, 6], count [N] int32): yolov5_official/utils.py:463-548."""
    _need_cuda(pred)
    lib = _ffi.lib()
    pred = pred.float().contiguous()
    N, nboxes, no = pred.shape
    dev = pred.device
    rows = torch.empty(N, max_box, 6, device=dev, dtype=torch.float32)
    count = torch.zeros(N, device=dev, dtype=torch.int32)
    if N == 0:
        return rows, count
    mask_ptr = None
    if classes:
        m = torch.zeros(no - 5, dtype=torch.uint8)
        m[torch.as_tensor(list(classes), dtype=torch.long)] = 1
        mask = m.to(dev)
        mask_ptr = mask.data_ptr()
    ws_bytes = lib.ydet_nms_cluster_diou_workspace_bytes(N, nboxes, no, max_box)
    ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
    with torch.cuda.device(dev):
        _ffi.check(lib.ydet_nms_cluster_diou(pred.data_ptr(), N, nboxes, no, float(conf_thres), float(iou_thres), int(max_box),
                                             int(bool(agnostic)), mask_ptr, rows.data_ptr(), count.data_ptr(), ws.data_ptr(),
                                             ws_bytes, _ffi.current_stream()), "ydet_nms_cluster_diou")
    return rows, count


def nms_perclass(boxes, scores, conf_thresh, nms_thresh, workspace_bytes=None):
    """boxes [N, n, 4], scores [N, n, nc] fp32 CUDA.
    Returns (keep [N, n] uint8, cls [N, n] int32, best [N, n] fp32): utils/utils.py:101-133.
    workspace_bytes: None = the full size (bit matrices for long class segments); "min" or a byte count in between
    leave some or all segments to the round-by-round walk (same result)."""
    _need_cuda(boxes, scores)
    lib = _ffi.lib()
    boxes = boxes.float().contiguous()
    scores = scores.float().contiguous()
    N, n, nc = scores.shape
    dev = boxes.device
    keep = torch.empty(N, n, device=dev, dtype=torch.uint8)
    cls = torch.empty(N, n, device=dev, dtype=torch.int32)
    best = torch.empty(N, n, device=dev, dtype=torch.float32)
    if N == 0 or n == 0:
        return keep, cls, best
    ws_bytes = lib.ydet_nms_perclass_workspace_bytes(N, n, nc)
    if workspace_bytes is not None:
        ws_min = lib.ydet_nms_perclass_workspace_bytes_min(N, n, nc)
        ws_bytes = ws_min if workspace_bytes == "min" else max(ws_min, min(ws_bytes, int(workspace_bytes)))
    ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
    with torch.cuda.device(dev):
        _ffi.check(lib.ydet_nms_perclass(boxes.data_ptr(), scores.data_ptr(), N, n, nc, float(conf_thresh),
                                         float(nms_thresh), keep.data_ptr(), cls.data_ptr(), best.data_ptr(),
                                         ws.data_ptr(), ws_bytes, _ffi.current_stream()), "ydet_nms_perclass")
    return keep, cls, best


def box_iou(box1, box2):
    """IoU matrix [n1, n2] of xyxy boxes (yolov5_official/utils.py:601-611)."""
    _need_cuda(box1, box2)
    lib = _ffi.lib()
    a = box1.float().contiguous()
    b = box2.float().contiguous()
    out = torch.empty(a.shape[0], b.shape[0], device=a.device, dtype=torch.float32)
    with torch.cuda.device(a.device):
        _ffi.check(lib.ydet_box_iou(a.data_ptr(), a.shape[0], b.data_ptr(), b.shape[0], out.data_ptr(),
                                    _ffi.current_stream()), "ydet_box_iou")
    return out


def process_batch(det, count, labels, label_start, iouv):
    """TP matrices of a batch in one launch (yolov5_official/utils.py:1103-1123 per image).
    det [B, max_det, 6] fp32, count [B] int32, labels [L, 5] (cls, xyxy) grouped by image, label_start [B + 1] int32,
    iouv [k] fp32, all CUDA.  Returns correct [B, max_det, k] bool (rows >= count are False)."""
    _need_cuda(det, count, label_start, iouv)
    lib = _ffi.lib()
    det = det.float().contiguous()
    count = count.to(torch.int32).contiguous()
    labels = labels.float().contiguous()
    label_start = label_start.to(torch.int32).contiguous()
    iouv = iouv.float().contiguous()
    B, max_det, _ = det.shape
    out = torch.empty(B, max_det, iouv.numel(), device=det.device, dtype=torch.uint8)
    if B == 0:
        return out.bool()
    assert label_start.numel() == B + 1 and count.numel() == B
    with torch.cuda.device(det.device):
        _ffi.check(lib.ydet_process_batch(det.data_ptr(), count.data_ptr(), B, max_det, labels.data_ptr(),
                                          label_start.data_ptr(), iouv.data_ptr(), iouv.numel(), out.data_ptr(),
                                          _ffi.current_stream()), "ydet_process_batch")
    return out.bool()


def voc_match(boxes, members, group_start, gt_boxes, gt_difficult, gt_start, ovthresh=0.5):
    """The matching loop of the VOC metric (data/vocapi_evaluator.py:284-318) for all (class, image) groups in one
    launch.  boxes [n, 4] float64; members [n] int32 (detection indices group by group, in visiting order);
    group_start / gt_start [G + 1] int32; gt_boxes [m, 4] float64; gt_difficult [m] uint8 -- all CUDA.
    Returns flags [n] uint8 per detection: 1 true positive, 2 false positive, 0 neither."""
    _need_cuda(boxes, members, group_start, gt_boxes, gt_difficult, gt_start)
    lib = _ffi.lib()
    boxes = boxes.to(torch.float64).contiguous()
    gt_boxes = gt_boxes.to(torch.float64).contiguous()
    members = members.to(torch.int32).contiguous()
    group_start = group_start.to(torch.int32).contiguous()
    gt_start = gt_start.to(torch.int32).contiguous()
    gt_difficult = gt_difficult.to(torch.uint8).contiguous()
    n, G = boxes.shape[0], group_start.numel() - 1
    assert members.numel() == n and gt_start.numel() == G + 1 and gt_boxes.shape[0] == gt_difficult.numel()
    flags = torch.zeros(n, device=boxes.device, dtype=torch.uint8)
    if n == 0 or G <= 0:
        return flags
    nbytes = lib.ydet_voc_match_workspace_bytes(n)
    ws = torch.empty((nbytes + 7) // 8, device=boxes.device, dtype=torch.float64)
    with torch.cuda.device(boxes.device):
        _ffi.check(lib.ydet_voc_match(boxes.data_ptr(), n, members.data_ptr(), group_start.data_ptr(), G,
                                      gt_boxes.data_ptr(), gt_difficult.data_ptr(), gt_start.data_ptr(), float(ovthresh),
                                      flags.data_ptr(), ws.data_ptr(), ws.numel() * 8, _ffi.current_stream()),
                   "ydet_voc_match")
    return flags


# ---- operators over the channels of every pixel ----------------------------------------------------------------------
# Tensors are [..., C]: any leading dimensions, the channels last (an NHWC map, or a channel slice of one).  Rows at one
# common distance are read where they lie; other strides, and types other than fp32 / bf16, are copied or refused.  What they
# cannot pass on is an error instead of a lost derivative: forward-mode tangents (_no_tangents), tracing (_as_rows), gradients of
# the 8-bit operators (_without_gradient).
MAX_ROW = 8192      # channels of a row that layer_norm and quantize_rows take


def _no_tangents(what, *ts):
    """Raises if one of the tensors carries a forward-mode tangent.  (Called where a dual level is open.)"""
    for t in ts:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{what} has no forward-mode derivative")


class _NoGradient(torch.autograd.Function):
    @staticmethod
    def forward(ctx, what, held, *inputs):
        ctx.what = what
        return held[0].detach()     # (an output of its own: as a tensor argument it would be a view that may not be changed in place)

    @staticmethod
    def backward(ctx, dy):
        raise NotImplementedError(f"{ctx.what} has no gradient: call it under torch.no_grad(), or on detached tensors")


def _without_gradient(what, y, *inputs):
    """y, in whose place in a recorded graph stands an error for the backward pass.  (Called where an input requires a gradient.)"""
    return _NoGradient.apply(what, (y,), *inputs) if torch.is_grad_enabled() else y


def _launch(dev, call, *args):
    """`call(*args, stream)` on torch's current stream of `dev`."""
    i = dev.index
    if torch._C._cuda_getDevice() == i:
        return call(*args, torch._C._cuda_getCurrentRawStream(i))
    with torch.cuda.device(i):
        return call(*args, torch._C._cuda_getCurrentRawStream(i))


def _as_rows(t, what):
    """(t or a copy, rows, distance of rows) of a [..., C] tensor."""
    shape = t.shape
    if not shape or not shape[-1]:
        raise ValueError(f"{what} needs at least one channel (shape {tuple(shape)})")
    C = shape[-1]
    if type(C) is not int:      # (a tensor while torch.jit.trace records, which would keep the result as a constant)
        raise RuntimeError(f"{what} cannot be traced")
    n = shape[0] if len(shape) == 2 else t.numel() // C
    if t.is_contiguous():
        return t, n, C
    if t.stride(-1) == 1 or C == 1:
        try:
            ld = t.view(-1, C).stride(0) if n > 1 else C
        except RuntimeError:
            ld = 0
        if C <= ld < 2 ** 31:
            return t, n, ld
    return t.contiguous(), n, C


def _params(C, dev, w, b):
    """The per-channel parameters (None allowed) as contiguous tensors of one type, and that type."""
    td = None
    want = (C,)
    for p in (w, b):
        if p is not None:
            if p.shape != want:
                raise ValueError(f"weight and bias have one value a channel: got {tuple(p.shape)} for {C} channels")
            if p.device != dev:
                raise RuntimeError(f"weight / bias on {p.device}, the input on {dev}")
            d = p.dtype
            if d is not torch.float32 and d is not torch.bfloat16:
                raise TypeError(f"unsupported dtype {d}")
            td = d if td is None or td is d else torch.float32
    if w is not None and (w.dtype is not td or not w.is_contiguous()):
        w = w.detach().to(td).contiguous()
    if b is not None and (b.dtype is not td or not b.is_contiguous()):
        b = b.detach().to(td).contiguous()
    return w, b, _ffi.BF16 if td is torch.bfloat16 else _ffi.F32


def _ptr(t):
    return None if t is None else t.data_ptr()


def _ln_forward(x, weight, bias, eps, stats):
    """(y, statistics): the means of all rows and then their reciprocal deviations in one fp32 buffer, or None."""
    if not x.is_cuda:
        _need_cuda(x)
    dt = _dt(x)
    x, n, ld = _as_rows(x, "layer_norm")
    C, dev = x.shape[-1], x.device
    w, b, pdt = _params(C, dev, weight, bias)
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    st = mean = rstd = None
    if stats:
        st = x.new_empty((2,) + x.shape[:-1], dtype=torch.float32)
        mean = st.data_ptr()
        rstd = mean + 4 * n
    d = _ffi.LayerNormDesc(x.data_ptr(), y.data_ptr(), w if w is None else w.data_ptr(), b if b is None else b.data_ptr(), mean, rstd,
                           n, C, ld, 0, C, 0, dt, pdt, eps)
    rc = _launch(dev, _ffi.lib().ydet_layer_norm, d)
    if rc:
        _ffi.check(rc, "ydet_layer_norm")
    return y, st


def layer_norm_forward(x, weight=None, bias=None, eps=1e-5):
    """Layer normalisation over the last dimension: (y, mean, rstd), y of x's dtype and shape, mean and rstd fp32 of
    x.shape[:-1].  weight, bias: [C] fp32 or bf16, or None.  The variance is an fp32 number: with eps = 0 a row whose variance
    is below 1.2e-38 counts as constant, and what is divided by its deviation is not finite; a row whose sum passes 3.4e38
    becomes NaN, one whose sum of squared differences does has rstd 0.  No autograd: y is not part of a recorded graph,
    layer_norm_backward takes the gradients."""
    if forward_ad._current_level >= 0:
        _no_tangents("layer_norm_forward", x, weight, bias)
    y, st = _ln_forward(x, weight, bias, eps, True)
    return y, st[0], st[1]


def _ln_backward(dy, x, mean, rstd, weight, need, bias_dtype):
    """mean, rstd: addresses."""
    lib = _ffi.lib()
    dt = _dt(x)
    x, n, ld = _as_rows(x, "layer_norm_backward")
    dy, _, dy_ld = _as_rows(dy, "layer_norm_backward")
    C, dev = x.shape[-1], x.device
    w, _, pdt = _params(C, dev, weight, None)
    wdt = torch.float32 if w is None else w.dtype
    if need[2] and bias_dtype is torch.float32 and wdt is not bias_dtype:     # (both gradients come in one type: the wider one)
        w, wdt, pdt = w.float(), bias_dtype, _ffi.F32
    dx = torch.empty_like(x, memory_format=torch.contiguous_format) if need[0] else None
    dw = x.new_empty(C, dtype=wdt) if need[1] else None
    db = x.new_empty(C, dtype=wdt) if need[2] else None
    ws, nbytes = None, 0
    if need[1] or need[2]:
        nbytes = lib.ydet_layer_norm_backward_workspace_bytes(n, C)
        ws = x.new_empty(nbytes, dtype=torch.uint8)
    d = _ffi.LayerNormGradDesc(dy.data_ptr(), x.data_ptr(), _ptr(dx), _ptr(w), mean, rstd, _ptr(dw), _ptr(db),
                               n, C, dy_ld, 0, ld, 0, C, 0, dt, pdt)
    rc = _launch(dev, lib.ydet_layer_norm_backward, d, _ptr(ws), nbytes)
    if rc:
        _ffi.check(rc, "ydet_layer_norm_backward")
    if dw is not None and weight is not None and weight.dtype != wdt:
        dw = dw.to(weight.dtype)
    if db is not None and bias_dtype is not None and bias_dtype != wdt:
        db = db.to(bias_dtype)
    return dx, dw, db


def layer_norm_backward(dy, x, mean, rstd, weight=None, need=(True, True, True), bias_dtype=None):
    """Gradients (dx, dweight, dbias) of layer_norm_forward from dy, its input and the statistics it returned.  `need` says
    which of the three are wanted (the others are None); dweight has the weight's dtype, dbias `bias_dtype` (default: the
    weight's; both fp32 without a weight).  Launches only: it can be captured into a graph."""
    _need_cuda(dy, x, mean, rstd)
    if dy.shape != x.shape or dy.dtype != x.dtype:
        raise ValueError(f"dy is {dy.dtype} {tuple(dy.shape)}, x is {x.dtype} {tuple(x.shape)}")
    if mean.shape != x.shape[:-1] or rstd.shape != x.shape[:-1] or mean.dtype != torch.float32 or rstd.dtype != torch.float32:
        raise ValueError("mean and rstd are the fp32 tensors that layer_norm_forward returned for x")
    if forward_ad._current_level >= 0:
        _no_tangents("layer_norm_backward", dy, x, mean, rstd, weight)
    if not x.device == dy.device == mean.device == rstd.device:
        raise RuntimeError("layer_norm_backward: tensors on different devices")
    mean, rstd = mean.contiguous(), rstd.contiguous()
    return _ln_backward(dy, x, mean.data_ptr(), rstd.data_ptr(), weight, need, bias_dtype)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, st = _ln_forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, st)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    def _gradients(ctx, dy):
        x, weight, st = ctx.saved_tensors
        if forward_ad._current_level >= 0:
            _no_tangents("layer_norm's backward pass", dy, x, weight)
        mean = st.data_ptr()
        return _ln_backward(dy, x, mean, mean + 2 * st.numel(), weight, ctx.needs_input_grad, ctx.bias_dtype) + (None,)

    _gradients_once = torch.autograd.function.once_differentiable(_gradients)

    @staticmethod
    def backward(ctx, dy):
        # (grad mode is on here only where a second derivative was asked for: its use is an error)
        return _LayerNorm._gradients_once(ctx, dy) if torch.is_grad_enabled() else _LayerNorm._gradients(ctx, dy)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Layer normalisation over the last dimension, differentiable in x, weight and bias (once).  A recorded graph cannot be
    captured (its leaves' gradients may belong to another stream): a captured training step calls layer_norm_forward and
    layer_norm_backward."""
    if forward_ad._current_level >= 0:
        _no_tangents("layer_norm", x, weight, bias)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        _need_cuda(x)
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("layer_norm: gradients are not recorded during graph capture; call layer_norm_forward and "
                               "layer_norm_backward there")
        if type(x.numel()) is not int:      # (as in _as_rows; inside apply sizes are plain numbers)
            raise RuntimeError("layer_norm cannot be traced")
        return _LayerNorm.apply(x, weight, bias, eps)
    return _ln_forward(x, weight, bias, eps, False)[0]


def _quantize(x, normalize, weight, bias, eps):
    if not x.is_cuda:
        _need_cuda(x)
    if forward_ad._current_level >= 0:
        _no_tangents("quantize_rows", x, weight, bias)
    dt = _dt(x)
    x, n, ld = _as_rows(x, "quantize_rows")
    C, dev, lead = x.shape[-1], x.device, x.shape[:-1]
    w, b, pdt = _params(C, dev, weight, bias)
    q_ld = (C + 15) // 16 * 16
    q = x.new_empty(*lead, q_ld, dtype=torch.int8)
    scale = x.new_empty(n, dtype=torch.float32)
    d = _ffi.QuantizeDesc(x.data_ptr(), q.data_ptr(), scale.data_ptr(), _ptr(w), _ptr(b), n, C, ld, 0, q_ld, dt, pdt, normalize, eps)
    rc = _launch(dev, _ffi.lib().ydet_quantize_rows_i8, d)
    if rc:
        _ffi.check(rc, "ydet_quantize_rows_i8")
    if len(lead) != 1:
        scale = scale.view(lead)
    if x.requires_grad or (weight is not None and weight.requires_grad) or (bias is not None and bias.requires_grad):
        scale = _without_gradient("quantize_rows", scale, x, weight, bias)
    return (q if q_ld == C else q[..., :C]), scale


def quantize_rows(x):
    """(q, scale): the rows of x [..., C] in 8 bits, q int8 of x's shape (its rows padded with zeros to 16 bytes in memory),
    scale fp32 of x.shape[:-1] with x ~ q * scale.  scale = max|x| / 127; q is the integer nearest x / scale, ties to even.
    A row with a NaN or an infinity has scale NaN and q = 0.  For inference: asking for a gradient through it is an error."""
    return _quantize(x, 0, None, None, 0.0)


def layer_norm_quantize(x, weight=None, bias=None, eps=1e-5):
    """quantize_rows(layer_norm(x, weight, bias, eps)) in one pass over x; the normalised values are not rounded in between.
    For inference, like quantize_rows."""
    return _quantize(x, 1, weight, bias, eps)


class LinearI8:
    """Weights of a token-wise linear layer (or 1x1 convolution) in 8 bits, laid out for matmul_i8: wq int8 [N, K], one fp32
    scale per output channel, an optional bias."""

    def __init__(self, wq, scale, bias=None):
        _need_cuda(wq, scale)
        if wq.dim() != 2 or wq.dtype != torch.int8 or wq.numel() == 0:
            raise ValueError(f"weights are int8 [N, K]: got {wq.dtype} {tuple(wq.shape)}")
        self.N, self.K = wq.shape
        dev = self.device = wq.device
        for t in (scale, bias):
            if t is not None and (t.shape != (self.N,) or t.device != dev or not t.is_floating_point()):
                raise ValueError(f"scale and bias are floating [{self.N}] tensors on {dev}")
        if self.K > 131071:
            raise ValueError(f"K = {self.K}: 32-bit sums hold products of up to 131071 terms")
        self.kp, self.n_pad = (self.K + 63) // 64 * 64, (self.N + 127) // 128 * 128
        self.w = torch.zeros(self.n_pad, self.kp, device=dev, dtype=torch.int8)
        self.w[:self.N, :self.K] = wq
        self.scale = torch.zeros(self.n_pad, device=dev)
        self.scale[:self.N] = scale.detach()
        self.bias = None
        if bias is not None:
            self.bias = torch.zeros(self.n_pad, device=dev)
            self.bias[:self.N] = bias.detach()

    @classmethod
    @torch.no_grad()
    def quantize(cls, weight, bias=None):
        """From floating weights [N, K] (or [N, K, 1, 1]): quantize_rows over every output channel's weights."""
        if weight.dim() == 4 and weight.shape[2:] == (1, 1):
            weight = weight[:, :, 0, 0]
        if weight.dim() != 2:
            raise ValueError(f"weights are [N, K] or [N, K, 1, 1]: got {tuple(weight.shape)}")
        q, scale = quantize_rows(weight.detach())
        return cls(q, scale, bias)


_ACTS = {"none": _ffi.ACT_NONE, "leaky": _ffi.ACT_LEAKY, "silu": _ffi.ACT_SILU}
_RES = {"after": _ffi.RES_AFTER_ACT, "before": _ffi.RES_BEFORE_ACT}


def _product(x, scale, n, ld, lin, act, slope, res, res_mode, out_dtype):
    """(output, descriptor, what it points to) of a product with `lin`; x, scale: addresses of n 8-bit rows and their scales."""
    if act not in _ACTS or res_mode not in _RES:
        raise ValueError(f"act {act!r} / res_mode {res_mode!r}: want one of {sorted(_ACTS)} / {sorted(_RES)}")
    if out_dtype == torch.bfloat16:
        odt = _ffi.BF16
    elif out_dtype == torch.float32:
        odt = _ffi.F32
    else:
        raise TypeError(f"unsupported dtype {out_dtype}")
    N, dev = lin.N, lin.device
    rmode, rptr, r_ld = _ffi.RES_NONE, None, 0
    if res is not None:
        if res.shape[-1:] != (N,) or res.numel() != n * N or res.dtype != out_dtype:
            raise ValueError(f"res is {out_dtype} of {n} rows of {N} channels: got {res.dtype} {tuple(res.shape)}")
        if res.device != dev:
            raise RuntimeError(f"res on {res.device}, the weights on {dev}")
        res, _, r_ld = _as_rows(res, "matmul_i8")
        rmode, rptr = _RES[res_mode], res.data_ptr()
    y = lin.w.new_empty(n, N, dtype=out_dtype)
    return y, _ffi.MatmulI8Desc(x, scale, lin.w.data_ptr(), lin.scale.data_ptr(), _ptr(lin.bias), rptr, y.data_ptr(), n, lin.K, N, lin.kp,
                                lin.n_pad, ld, 0, N, 0, r_ld, 0, _ACTS[act], slope, rmode, odt), res


def matmul_i8(q, scale, lin, act="none", slope=0.1, res=None, res_mode="after", out_dtype=torch.bfloat16):
    """act(q . lin.w^T * scale * lin.scale + lin.bias), [..., N] of out_dtype (bf16 or fp32), from int8 rows q [..., K] and
    their scales [...] (quantize_rows).  act: "none", "leaky" (negative slope `slope`), "silu".  res [..., N] of out_dtype is
    added after or before the activation (res_mode).  The sums are exact integers.  For inference: asking for a gradient
    through it is an error."""
    if not (q.is_cuda and scale.is_cuda):
        _need_cuda(q, scale)
    if forward_ad._current_level >= 0:
        _no_tangents("matmul_i8", scale, res)
    K, shape = lin.K, q.shape
    if q.dtype != torch.int8 or len(shape) == 0 or shape[-1] != K:
        raise ValueError(f"q is int8 [..., {K}]: got {q.dtype} {tuple(shape)}")
    lead = shape[:-1]
    if scale.shape != lead or scale.dtype != torch.float32:
        raise ValueError(f"scale is fp32 {tuple(lead)}: got {scale.dtype} {tuple(scale.shape)}")
    if res is not None and res.shape[:-1] != lead:
        raise ValueError(f"res is [..., {lin.N}] with q's leading dimensions {tuple(lead)}: got {tuple(res.shape)}")
    dev = q.device
    if dev != lin.device or dev != scale.device:
        raise RuntimeError("matmul_i8: tensors on different devices")
    q, n, ld = _as_rows(q, "matmul_i8")
    # the library may read a row's last piece up to its 16-byte border: a view whose storage ends before that is copied
    if ld > 1 << 23 or (K % 16 and ld % 16 == 0 and n and q.data_ptr() % 16 == 0 and
                        q.storage_offset() + (n - 1) * ld + (K + 15) // 16 * 16 > q.untyped_storage().nbytes()):
        q, ld = q.clone(memory_format=torch.contiguous_format), K
    if not scale.is_contiguous():
        scale = scale.contiguous()
    at = q.data_ptr()       # (0 without rows)
    y, d, keep = _product(at, scale.data_ptr(), n, ld, lin, act, slope, res, res_mode, out_dtype)
    lib = _ffi.lib()
    ws, nbytes = None, 0
    if (ld | at) % 4:
        nbytes = lib.ydet_matmul_i8_workspace_bytes(d)
        ws = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    rc = _launch(dev, lib.ydet_matmul_i8, d, _ptr(ws), nbytes)
    if rc:
        _ffi.check(rc, "ydet_matmul_i8")
    if len(lead) != 1:
        y = y.view(lead + (lin.N,))
    if scale.requires_grad or (res is not None and res.requires_grad):
        return _without_gradient("matmul_i8", y, scale, res)
    return y


def linear_i8(x, lin, act="none", slope=0.1, res=None, res_mode="after", out_dtype=None):
    """matmul_i8 of a floating map x [..., K], whose rows are quantised (quantize_rows) on the way; out_dtype defaults to x's.
    The same bits as the two calls; K up to MAX_ROW.  For inference: asking for a gradient through it is an error."""
    if not x.is_cuda:
        _need_cuda(x)
    if forward_ad._current_level >= 0:
        _no_tangents("linear_i8", x, res)
    K, shape = lin.K, x.shape
    if shape[-1:] != (K,):
        raise ValueError(f"x is [..., {K}]: got {tuple(shape)}")
    lead = shape[:-1]
    if res is not None and res.shape[:-1] != lead:
        raise ValueError(f"res is [..., {lin.N}] with x's leading dimensions {tuple(lead)}: got {tuple(res.shape)}")
    dev = x.device
    if dev != lin.device:
        raise RuntimeError("linear_i8: tensors on different devices")
    lib = _ffi.lib()
    dt = _dt(x)
    x, n, ld = _as_rows(x, "linear_i8")
    y, d, keep = _product(None, None, n, 0, lin, act, slope, res, res_mode, x.dtype if out_dtype is None else out_dtype)
    src = _ffi.QuantizeDesc(x.data_ptr(), None, None, None, None, n, K, ld, 0, 0, dt, _ffi.F32, 0, 0.0)
    nbytes = lib.ydet_linear_i8_workspace_bytes(src, d)
    ws = x.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    rc = _launch(dev, lib.ydet_linear_i8, src, d, _ptr(ws), nbytes)
    if rc:
        _ffi.check(rc, "ydet_linear_i8")
    if len(lead) != 1:
        y = y.view(lead + (lin.N,))
    if x.requires_grad or (res is not None and res.requires_grad):
        return _without_gradient("linear_i8", y, x, res)
    return y
