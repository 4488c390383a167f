"""Operator-level entry points of the detection graph, one per native operator the
reference graph calls (symbol/faster_rcnn.py:98-103) plus the detector tail
(detection.py:47-58).  NumPy in -> NumPy out, torch in -> torch (device) out."""
import ctypes as C
from typing import NamedTuple

import numpy as np
import torch

from . import _lib, runtime
from .symbol.config import config as _global_config


def make_proposal_cfg(feature_stride=16, scales=(4, 8, 16, 32), ratios=(0.5, 1, 2), rpn_pre_nms_top_n=None,
                      rpn_post_nms_top_n=None, threshold=None, rpn_min_size=None, box_f64=True):
    """fd_proposal_cfg from the keyword names of ``mx.symbol.contrib.Proposal``; values left
    at None are read from the global config, as symbol/faster_rcnn.py:100-102 does."""
    T = _global_config.TEST
    cfg = _lib.ProposalCfg()
    cfg.feat_stride = int(feature_stride)
    scales, ratios = list(scales), list(ratios)
    if not (0 < len(scales) <= 8 and 0 < len(ratios) <= 8):
        raise ValueError("between 1 and 8 scales and ratios are supported")
    cfg.num_scales, cfg.num_ratios = len(scales), len(ratios)
    for i, s in enumerate(scales):
        cfg.scales[i] = float(s)
    for i, r in enumerate(ratios):
        cfg.ratios[i] = float(r)
    cfg.pre_nms_top_n = int(T.RPN_PRE_NMS_TOP_N if rpn_pre_nms_top_n is None else rpn_pre_nms_top_n)
    cfg.post_nms_top_n = int(T.RPN_POST_NMS_TOP_N if rpn_post_nms_top_n is None else rpn_post_nms_top_n)
    cfg.nms_thresh = float(T.RPN_NMS_THRESH if threshold is None else threshold)
    cfg.min_size = float(T.RPN_MIN_SIZE if rpn_min_size is None else rpn_min_size)
    cfg.box_f64 = 1 if box_f64 else 0
    return cfg


def proposal(cls_prob, bbox_pred, im_info, output_score=False, return_counts=False, **kwargs):
    """``contrib.Proposal``: cls_prob [B,2A,H,W], bbox_pred [B,4A,H,W], im_info [B,3] ->
    rois [B*post_n, 5].  Raises ValueError on NaN input like the reference operator
    (proposal.py:47-51).  ``kwargs`` are those of :func:`make_proposal_cfg`."""
    as_np = not isinstance(cls_prob, torch.Tensor)
    cfg = make_proposal_cfg(**kwargs)
    if cfg.post_nms_top_n <= 0:
        raise ValueError("rpn_post_nms_top_n must be positive (the output has a fixed number of rows)")
    B, C2, H, W = (int(v) for v in cls_prob.shape)
    A = cfg.num_scales * cfg.num_ratios
    if C2 != 2 * A or tuple(int(v) for v in bbox_pred.shape[:2]) != (B, 4 * A):
        raise ValueError("proposal: cls_prob [B,%d,H,W] and bbox_pred [B,%d,H,W] expected" % (2 * A, 4 * A))
    ctx = runtime.context()
    cls_d = runtime.to_device(cls_prob, torch.float32)
    box_d = runtime.to_device(bbox_pred, torch.float32)
    if tuple(box_d.shape[2:]) != (H, W):          # clip_pad (processing.py:99-112)
        box_d = box_d[:, :, :H, :W].contiguous()
    info = np.ascontiguousarray(np.asarray(im_info.cpu() if isinstance(im_info, torch.Tensor) else im_info,
                                           dtype=np.float32).reshape(B, 3))
    rois = runtime.empty((B * cfg.post_nms_top_n, 5), torch.float32)
    scores = runtime.empty((B * cfg.post_nms_top_n,), torch.float32)
    counts = runtime.empty((B, 3), torch.int32)
    nan_flag = runtime.empty((1,), torch.int32)
    _lib.check(_lib.lib().fd_proposal(ctx.handle, C.byref(cfg), runtime.ptr(cls_d), runtime.ptr(box_d),
                                      info.ctypes.data_as(_lib.c_f32p), B, H, W, runtime.ptr(rois),
                                      runtime.ptr(scores), runtime.ptr(counts), runtime.ptr(nan_flag),
                                      runtime.stream_ptr()))
    if int(nan_flag.item()) != 0:
        raise ValueError("there is nan in input scores or bbox_deltas")
    out = [rois.cpu().numpy() if as_np else rois]
    if output_score:
        s = scores.reshape(-1, 1)
        out.append(s.cpu().numpy() if as_np else s)
    if return_counts:
        out.append(counts.cpu().numpy())
    return out[0] if len(out) == 1 else tuple(out)


def roi_pooling(data, rois, pooled_size=(7, 7), spatial_scale=0.0625):
    """``mx.symbol.ROIPooling``: data [B,C,H,W], rois [R,5] -> [R,C,ph,pw]."""
    as_np = not isinstance(data, torch.Tensor)
    B, Cc, H, W = (int(v) for v in data.shape)
    R = int(rois.shape[0])
    ph, pw = int(pooled_size[0]), int(pooled_size[1])
    ctx = runtime.context()
    d = runtime.to_device(data, torch.float32)
    r = runtime.to_device(rois, torch.float32)
    out = runtime.empty((R, Cc, ph, pw), torch.float32)
    _lib.check(_lib.lib().fd_roipool(ctx.handle, runtime.ptr(d), B, Cc, H, W, runtime.ptr(r), R, ph, pw,
                                     float(spatial_scale), runtime.ptr(out), runtime.stream_ptr()))
    return out.cpu().numpy() if as_np else out


def postprocess(rois, scores, bbox_deltas, im_shape, thresh=0.8, nms_thresh=0.3, do_round=True):
    """Detector tail (detection.py:47-58): rois [R,4], scores [R,2], bbox_deltas [R,8] -> dets [n,5] float32."""
    as_np = not isinstance(rois, torch.Tensor)
    R = int(rois.shape[0])
    if R == 0:
        return np.zeros((0, 5), np.float32) if as_np else torch.zeros((0, 5))
    ctx = runtime.context()
    r = runtime.to_device(rois, torch.float32)
    s = runtime.to_device(scores, torch.float32)
    d = runtime.to_device(bbox_deltas, torch.float32)
    dets = runtime.empty((R, 5), torch.float32)
    n = runtime.empty((1,), torch.int32)
    _lib.check(_lib.lib().fd_postprocess(ctx.handle, runtime.ptr(r), runtime.ptr(s), runtime.ptr(d), R,
                                         int(im_shape[0]), int(im_shape[1]), float(thresh), float(nms_thresh),
                                         1 if do_round else 0, runtime.ptr(dets), runtime.ptr(n),
                                         runtime.stream_ptr()))
    k = int(n.item())
    out = dets[:k]
    return out.cpu().numpy() if as_np else out


def conv2d(x, weight, stride=1, pad=0, bias=None, pre_scale=None, pre_shift=None, relu=False, residual=None,
           precision="f32"):
    """``mx.sym.Convolution`` fused with its neighbours (see fd_conv2d in facedet.h).

    x [B,H,W,Cin] channels-last, weight [Cout,Cin,kh,kw] (MXNet layout); returns y [B,Ho,Wo,Cout].
    y = relu?(conv(relu(x*pre_scale+pre_shift)?) + bias?) + residual?"""
    as_np = not isinstance(x, torch.Tensor)
    B, H, W, Cin = (int(v) for v in x.shape)
    Cout, Cin_w, kh, kw = (int(v) for v in weight.shape)
    if Cin_w != Cin:
        raise ValueError("conv2d: weight expects %d input channels, x has %d" % (Cin_w, Cin))
    Ho = (H + 2 * pad - kh) // stride + 1
    Wo = (W + 2 * pad - kw) // stride + 1
    ctx = runtime.context()
    dev = lambda a: None if a is None else runtime.to_device(a, torch.float32)
    xd, wd, bd, sd, hd, rd = dev(x), dev(weight), dev(bias), dev(pre_scale), dev(pre_shift), dev(residual)
    y = runtime.empty((B, Ho, Wo, Cout), torch.float32)
    if precision in ("winograd", "winograd4"):
        # float32, Winograd F(2x2,3x3) or F(4x4,3x3): the 3x3 / stride 1 / pad 1 case without prologue or residual
        if (kh, kw, int(stride), int(pad)) != (3, 3, 1, 1) or sd is not None or hd is not None or rd is not None:
            raise ValueError("conv2d: the Winograd form is the plain 3x3, stride 1, pad 1 convolution")
        _lib.check(_lib.lib().fd_conv2d_winograd(ctx.handle, runtime.ptr(xd), B, H, W, Cin, runtime.ptr(wd), Cout,
                                                  runtime.ptr(bd), 1 if relu else 0, 4 if precision == "winograd4" else 2,
                                                  runtime.ptr(y), runtime.stream_ptr()))
        return y.cpu().numpy() if as_np else y
    fn = {"f32": _lib.lib().fd_conv2d, "f16x3": _lib.lib().fd_conv2d_f16x3, "bf16x3": _lib.lib().fd_conv2d_bf16x3}[precision]
    _lib.check(fn(ctx.handle, runtime.ptr(xd), B, H, W, Cin, runtime.ptr(wd), Cout, kh, kw,
                  int(stride), int(pad), runtime.ptr(bd), runtime.ptr(sd), runtime.ptr(hd),
                  1 if relu else 0, runtime.ptr(rd), runtime.ptr(y), runtime.stream_ptr()))
    return y.cpu().numpy() if as_np else y


def resize_bilinear(im, fx, fy):
    """``cv2.resize(im, None, None, fx=fx, fy=fy, interpolation=cv2.INTER_LINEAR)`` for uint8 images
    [H,W,C] or batches [B,H,W,C] (C <= 4)."""
    as_np = not isinstance(im, torch.Tensor)
    single = im.ndim == 3
    t = runtime.to_device(im, torch.uint8)
    if single:
        t = t.unsqueeze(0)
    B, H, W, Cc = (int(v) for v in t.shape)
    dh, dw = C.c_int32(0), C.c_int32(0)
    _lib.check(_lib.lib().fd_resize_dims(H, W, float(fx), float(fy), C.byref(dh), C.byref(dw)))
    out = runtime.empty((B, dh.value, dw.value, Cc), torch.uint8)
    ctx = runtime.context()
    _lib.check(_lib.lib().fd_resize_u8(ctx.handle, runtime.ptr(t), B, H, W, Cc, float(fx), float(fy),
                                       runtime.ptr(out), dh.value, dw.value, runtime.stream_ptr()))
    if single:
        out = out[0]
    return out.cpu().numpy() if as_np else out


def crop_resize_pad(frame, boxes, des_size=(112, 112), tiles=True):
    """``Function.stick_boxes`` + ``Function.resize_pad`` (code/common/Function.py:49-70,95-113) for
    all boxes of one uint8 frame [H,W,C] in one launch.  ``boxes`` [n,>=4] (x1,y1,x2,y2,...):
    detections or tracker rows.  Returns (tiles uint8 [n,des_h,des_w,C], rects int32 [n,4]) as
    NumPy arrays for a NumPy frame, device tensors otherwise; ``tiles=False`` computes the
    rectangles only."""
    as_np = not isinstance(frame, torch.Tensor)
    f = runtime.to_device(frame, torch.uint8)
    H, W, Cc = (int(v) for v in f.shape)
    b = runtime.to_device(boxes if isinstance(boxes, torch.Tensor) else np.asarray(boxes, dtype=np.float64),
                          torch.float64)
    if b.dim() != 2 or b.shape[1] < 4:
        raise ValueError("boxes must be [n, >=4]")
    n = int(b.shape[0])
    dh, dw = int(des_size[0]), int(des_size[1])
    out = runtime.empty((n, dh, dw, Cc), torch.uint8) if tiles else None
    rects = runtime.empty((n, 4), torch.int32)
    ctx = runtime.context()
    _lib.check(_lib.lib().fd_crop_resize_pad(ctx.handle, runtime.ptr(f), H, W, Cc, runtime.ptr(b), int(b.shape[1]), n,
                                             dh, dw, runtime.ptr(out) if tiles else None, runtime.ptr(rects),
                                             runtime.stream_ptr()))
    if as_np:
        return (out.cpu().numpy() if tiles else None), rects.cpu().numpy()
    return out, rects


def crop_rects(boxes, height, width):
    """The padded, clamped slice bounds of ``Function.stick_boxes`` (code/common/Function.py:53-64)
    for boxes [n,>=4] in a frame of the given size: (None, int32 [n,4] NumPy array)."""
    b = runtime.to_device(boxes if isinstance(boxes, torch.Tensor) else np.asarray(boxes, dtype=np.float64),
                          torch.float64)
    n = int(b.shape[0])
    rects = runtime.empty((n, 4), torch.int32)
    ctx = runtime.context()
    _lib.check(_lib.lib().fd_crop_resize_pad(ctx.handle, None, int(height), int(width), 3, runtime.ptr(b),
                                             int(b.shape[1]), n, 1, 1, None, runtime.ptr(rects),
                                             runtime.stream_ptr()))
    return None, rects.cpu().numpy()


# ---------------------------------------------------------------------------------------------------------
# Expert block: the operators of a residual block whose products are split over experts, on rows [T, width]
# (rois, or positions of a channels-last map).  float32, float16 and bfloat16 rows (anything else is converted
# to float32), float32 arithmetic.
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_ACTS = {None: 0, "relu": 1, "silu": 2, "gelu": 3}
_GATE_ACTS = {None: 0, "sigmoid": 1, "tanh": 2}
_NP_TYPES = {"float32": torch.float32, "float16": torch.float16}


def _row_type(a):
    t = a.dtype if isinstance(a, torch.Tensor) else _NP_TYPES.get(np.asarray(a).dtype.name)
    return t if t in _DTYPES else torch.float32


_INT_MAX = 2 ** 31 - 1          # sizes that the library takes as an int would arrive there as others if they had more bits


def _too_large(name, size):
    raise ValueError("%s: sizes of at most %d, not %d" % (name, _INT_MAX, size))


def _rows(a, index, name, dtype=None):
    """A [rows, width] tensor on the GPU in its own type, or in ``dtype`` (another of the three types is refused)."""
    if a.ndim != 2:
        raise ValueError("%s must be [rows, width], not %d-dimensional" % (name, a.ndim))
    return _typed(a, index, name, dtype)


def _typed(a, index, name, dtype=None):
    if isinstance(a, torch.Tensor) and a.dtype is dtype:
        return runtime.rows_to_device(a, dtype, index)
    t = _row_type(a)
    if dtype is not None and t != dtype:
        if (a.dtype if isinstance(a, torch.Tensor) else _NP_TYPES.get(a.dtype.name)) in _DTYPES:
            raise ValueError("%s is %s, %s expected" % (name, t, dtype))
        t = dtype
    return runtime.rows_to_device(a, t, index)


def _ints(a, index, name):
    """int32 indices on the GPU; a wider type is refused, since a conversion could wrap."""
    if a.dtype is not torch.int32 and str(a.dtype) != "int32":
        raise ValueError("%s must be int32, not %s" % (name, a.dtype))
    return runtime.rows_to_device(a, torch.int32, index)


def _params(a, index, name, width):
    if a is None:
        return None
    if tuple(a.shape) != (width,):
        raise ValueError("%s must have shape (%d,), not %s" % (name, width, tuple(a.shape)))
    return runtime.rows_to_device(a, torch.float32, index)


def _ptr(t):
    return None if t is None else t.data_ptr()


class ExpertRoute(NamedTuple):
    """What :func:`expert_route` returns (see there)."""
    weights: object
    experts: object
    slots: object
    offsets: object
    rows: object


def expert_route(logits, top_k, mask=None, normalize=True):
    """Route of rows to experts.  logits [T, E] -> ExpertRoute of

    * weights [T, k] float32: softmax over the row's choices, or with ``normalize=False`` over all E experts;
    * experts [T, k] int32: the row's k largest logits, descending, equal ones by ascending expert;
    * slots [T, k] int32: the position of each choice when all are sorted by expert, then by row;
    * offsets [E + 1] int32: expert e has the slots offsets[e] .. offsets[e + 1] - 1;
    * rows [T * k] int32: the row of each slot, -1 from offsets[E] on.

    A logit of -inf or NaN is never chosen, and rows where ``mask`` [T] (bool or uint8) is false choose nothing; a
    choice that is not made is -1 with weight 0.  At most 512 experts and 16 choices."""
    as_np = not isinstance(logits, torch.Tensor)
    index, stream = runtime.current()
    x = _rows(logits, index, "logits")
    T, E = x.shape
    if E > _INT_MAX:
        _too_large("logits", E)
    k = int(top_k)
    if not 0 < k <= E:
        raise ValueError("top_k must be between 1 and the %d experts, not %d" % (E, k))
    if mask is not None:
        if tuple(mask.shape) != (T,) or str(mask.dtype).split(".")[-1] not in ("bool", "uint8"):
            raise ValueError("mask must be bool or uint8 of shape (%d,)" % T)
        mask = runtime.rows_to_device(mask, torch.bool, index)
    L = _lib.lib()
    weights, chosen, slots = x.new_empty((T, k), dtype=torch.float32), x.new_empty((T, k), dtype=torch.int32), x.new_empty((T, k), dtype=torch.int32)
    offsets, source = x.new_empty((E + 1,), dtype=torch.int32), x.new_empty((T * k,), dtype=torch.int32)
    nbytes = L.fd_expert_route_workspace(T, E)
    work = x.new_empty((nbytes,), dtype=torch.uint8) if nbytes else None
    _lib.check(L.fd_expert_route(x.data_ptr(), _DTYPES[x.dtype], T, E, k, _ptr(mask), 1 if normalize else 0, weights.data_ptr(),
                                 chosen.data_ptr(), slots.data_ptr(), offsets.data_ptr(), source.data_ptr(), _ptr(work), nbytes,
                                 stream))
    out = ExpertRoute(weights, chosen, slots, offsets, source)
    return ExpertRoute(*(t.cpu().numpy() for t in out)) if as_np else out


def expert_linear(x, weight, offsets, rows=None, bias=None, activation=None, gated=False):
    """Matrix products grouped by expert: x [T, K], weight [E, N, K] -> y [S, N], S = len(rows), or T without ``rows``.

    Slot s with offsets[e] <= s < offsets[e + 1] is expert e's: y[s] = act(x[rows[s]] @ weight[e].T + bias[e]), or
    of x[s] without ``rows`` (x is in slot order then).  ``activation``: None, "relu", "silu" or "gelu" (the erf form).
    ``gated``: weight [E, 2N, K] and bias [E, 2N] hold two halves and y[s] = act(first half) * second half.
    ``offsets`` and ``rows`` are int32 as :func:`expert_route` gives them; slots from offsets[E] on become zeros, an
    index of ``rows`` outside x reads as a row of zeros.  x, weight and bias are of one type, and so is y."""
    as_np = not isinstance(x, torch.Tensor)
    index, stream = runtime.current()
    x = _rows(x, index, "x")
    T, K = x.shape
    if weight.ndim != 3 or weight.shape[2] != K:
        raise ValueError("weight must be [experts, outputs, %d], not %s" % (K, tuple(weight.shape)))
    E, n, _ = weight.shape
    if K > _INT_MAX or E > _INT_MAX or n > _INT_MAX:
        _too_large("weight", max(K, E, n))
    w = _typed(weight, index, "weight", x.dtype)
    if gated and n % 2:
        raise ValueError("a gated weight has two halves of rows, not %d rows" % n)
    N = n // 2 if gated else n
    if activation not in _ACTS:
        raise ValueError("unknown activation %r" % (activation,))
    if tuple(offsets.shape) != (E + 1,):
        raise ValueError("offsets must have shape (%d,), not %s" % (E + 1, tuple(offsets.shape)))
    o = _ints(offsets, index, "offsets")
    if rows is not None:
        if rows.ndim != 1:
            raise ValueError("rows must be one-dimensional")
        rows = _ints(rows, index, "rows")
    if bias is not None:
        if tuple(bias.shape) != (E, n):
            raise ValueError("bias must have shape (%d, %d), not %s" % (E, n, tuple(bias.shape)))
        bias = _typed(bias, index, "bias", x.dtype)
    S = T if rows is None else rows.shape[0]
    y = x.new_empty((S, N))
    _lib.check(_lib.lib().fd_expert_linear(x.data_ptr(), _DTYPES[x.dtype], T, K, w.data_ptr(), E, N, o.data_ptr(), _ptr(rows), S,
                                           _ptr(bias), _ACTS[activation], 1 if gated else 0, y.data_ptr(), stream))
    return y.cpu().numpy() if as_np else y


def _slots_weights(slots, weights, index, rows):
    if slots.ndim != 2 or tuple(weights.shape) != tuple(slots.shape) or (rows is not None and slots.shape[0] != rows):
        raise ValueError("slots and weights must both be [rows, k], not %s and %s" % (tuple(slots.shape), tuple(weights.shape)))
    if not 0 < slots.shape[1] <= _INT_MAX:
        if slots.shape[1]:
            _too_large("slots", slots.shape[1])
        raise ValueError("slots has no columns")
    return _ints(slots, index, "slots"), runtime.rows_to_device(weights, torch.float32, index)


def expert_combine(y, slots, weights):
    """Weighted sum of a row's expert outputs: y [S, N], slots / weights [T, k] -> out [T, N],
    out[t] = sum over j of weights[t, j] * y[slots[t, j]] in the order of j.  A slot outside y (-1) adds nothing."""
    as_np = not isinstance(y, torch.Tensor)
    index, stream = runtime.current()
    y = _rows(y, index, "y")
    s, w = _slots_weights(slots, weights, index, None)
    T, k = s.shape
    S, N = y.shape
    if N > _INT_MAX:
        _too_large("y", N)
    out = y.new_empty((T, N))
    _lib.check(_lib.lib().fd_expert_combine(y.data_ptr(), _DTYPES[y.dtype], S, N, s.data_ptr(), w.data_ptr(), T, k,
                                            out.data_ptr(), stream))
    return out.cpu().numpy() if as_np else out


def _norm_kind(kind):
    if kind not in ("rms", "layer"):
        raise ValueError("kind must be 'rms' or 'layer', not %r" % (kind,))
    return 1 if kind == "layer" else 0


def block_norm(x, weight, bias=None, kind="rms", eps=1e-6, dtype=None):
    """The norm before a block: x [T, N] -> u [T, N] = x / sqrt(mean(x^2) + eps) * weight + bias, for ``kind="layer"`` of
    x - mean(x).  weight and bias are float32 [N].  u has x's type; a float32 x (a residual stream held in float32 beside 16-bit
    blocks) may give u in the torch type ``dtype``, rounded once, at the end."""
    as_np = not isinstance(x, torch.Tensor)
    index, stream = runtime.current()
    x = _rows(x, index, "x")
    T, N = x.shape
    if N > _INT_MAX:
        _too_large("x", N)
    weight, bias = _params(weight, index, "weight", N), _params(bias, index, "bias", N)
    t = _DTYPES[x.dtype]
    if dtype is None or dtype is x.dtype:
        u, th = torch.empty_like(x), t
    elif dtype not in _DTYPES or t != 0 or (as_np and dtype is torch.bfloat16):          # NumPy has no bfloat16
        raise ValueError("u of %s rows cannot be %s" % (x.dtype, dtype))
    else:
        u, th = torch.empty_like(x, dtype=dtype), _DTYPES[dtype]
    a = _lib.NormArgs(x=x.data_ptr(), u=u.data_ptr(), pre_weight=_ptr(weight), pre_bias=_ptr(bias), rows=T, width=N, x_dtype=t, h_dtype=th,
                      layer=_norm_kind(kind), eps=float(eps))
    _lib.check(_lib.lib().fd_residual_norm(C.byref(a), stream))
    return u.cpu().numpy() if as_np else u


def residual_norm(x, h, post_weight=None, post_bias=None, gate=None, gate_activation=None, scale=1.0, pre_weight=None, pre_bias=None,
                  kind="rms", eps=1e-6, slots=None, weights=None):
    """The end of a residual block and the start of the next: x [T, N] (the residual stream), h (the block's output) ->
    (x', u), or x' alone without ``pre_weight``:

        x' = x + scale * act(gate) * norm(h; post_weight, post_bias)        (``post_weight=None``: h as it is)
        u  = norm(x'; pre_weight, pre_bias)

    with the norms of :func:`block_norm`.  h is [T, N], or with ``slots`` and ``weights`` [T, k] an expert block's
    [S, N], whose sum (:func:`expert_combine`) is formed on the way.  ``gate``: [N], or [G, N] with a row for each T / G
    consecutive rows (one per frame, or with G = T one per row), float32 or of h's type; ``gate_activation``: None, "sigmoid"
    or "tanh".  x is of h's type or float32; x' has x's type, u has h's.  Weights and biases are float32 [N]."""
    as_np = not isinstance(x, torch.Tensor)
    index, stream = runtime.current()
    h = _rows(h, index, "h")
    x = _rows(x, index, "x", None if _row_type(x) == torch.float32 else h.dtype)
    T, N = x.shape
    if N > _INT_MAX:
        _too_large("x", N)
    if h.shape[1] != N or (slots is None and h.shape[0] != T):
        raise ValueError("h is %s, x is %s" % (tuple(h.shape), tuple(x.shape)))
    if (slots is None) != (weights is None):
        raise ValueError("slots and weights come together")
    if gate_activation not in _GATE_ACTS:
        raise ValueError("unknown gate activation %r" % (gate_activation,))
    if gate_activation is not None and gate is None:
        raise ValueError("gate_activation without a gate")
    if (post_bias is not None and post_weight is None) or (pre_bias is not None and pre_weight is None):
        raise ValueError("a bias needs its weight")
    a = _lib.NormArgs(x=x.data_ptr(), h=h.data_ptr(), rows=T, h_rows=h.shape[0], width=N, x_dtype=_DTYPES[x.dtype],
                      h_dtype=_DTYPES[h.dtype], layer=_norm_kind(kind), scale=float(scale), eps=float(eps))
    if slots is not None:
        slots, weights = _slots_weights(slots, weights, index, T)
        a.slots, a.weights, a.k = slots.data_ptr(), weights.data_ptr(), slots.shape[1]
    if gate is not None:
        if gate.ndim not in (1, 2) or gate.shape[-1] != N or (gate.ndim == 2 and T and (gate.shape[0] == 0 or T % gate.shape[0])):
            raise ValueError("gate must be [%d] or [G, %d] with G a divisor of %d rows, not %s" % (N, N, T, tuple(gate.shape)))
        gate = runtime.rows_to_device(gate, h.dtype if _row_type(gate) == h.dtype else torch.float32, index)
        a.gate, a.gate_rows = gate.data_ptr(), gate.shape[0] if gate.ndim == 2 else 1
        a.gate_dtype, a.gate_act = _DTYPES[gate.dtype], _GATE_ACTS[gate_activation]
    post_weight, post_bias = _params(post_weight, index, "post_weight", N), _params(post_bias, index, "post_bias", N)
    pre_weight, pre_bias = _params(pre_weight, index, "pre_weight", N), _params(pre_bias, index, "pre_bias", N)
    a.post_weight, a.post_bias, a.pre_weight, a.pre_bias = _ptr(post_weight), _ptr(post_bias), _ptr(pre_weight), _ptr(pre_bias)
    new = torch.empty_like(x)
    u = h.new_empty((T, N)) if pre_weight is not None else None
    a.x_out, a.u = new.data_ptr(), _ptr(u)
    _lib.check(_lib.lib().fd_residual_norm(C.byref(a), stream))
    if as_np:
        new, u = new.cpu().numpy(), None if u is None else u.cpu().numpy()
    return new if u is None else (new, u)
