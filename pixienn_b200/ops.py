"""The epilogue operators on torch CUDA tensors.

Thin argument marshalling over the C ABI (``include/pxe.h``): torch supplies device memory and
the current stream, every computation runs in ``libpxe.so``.  A tensor argument may be a channel
slice of a wider NCHW buffer (``buf[:, 64:192]``): its batch stride is passed through, which is
how producers write straight into route (concat) buffers.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional, Sequence

import numpy as np
import torch

from . import capi
from .capi import ACT, PxeError  # noqa: F401  (re-exported)

DET_DTYPE = np.dtype([("x", "f4"), ("y", "f4"), ("w", "f4"), ("h", "f4"), ("prob", "f4"),
                      ("class_id", "i4"), ("batch_id", "i4"), ("source", "i4")])


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _act(a) -> int:
    return ACT[a] if isinstance(a, str) else int(a)


def _check_device(index: int, name: str) -> None:
    """The library launches on the calling thread's current device and on torch's current stream of that
    device, so a tensor of another GPU must not reach it: without peer access the kernel would fault, with it
    the work would silently run on the wrong GPU.  Callers select the device first (``torch.cuda.device``;
    Runner and PipelinedPredictor do it themselves)."""
    cur = torch.cuda.current_device()
    if index != cur:
        raise ValueError(f"{name} lives on cuda:{index} but the current device is cuda:{cur}; "
                         f"wrap the call in torch.cuda.device({index})")


def _check_f32_cuda(t: torch.Tensor, name: str) -> None:
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype == torch.float32):
        raise TypeError(f"{name} must be a float32 CUDA tensor")
    _check_device(t.device.index, name)


def _slot(t: Optional[torch.Tensor], name: str):
    """(pointer, batch stride) of a 4-D NCHW tensor whose per-image block is dense."""
    if t is None:
        return None, 0
    _check_f32_cuda(t, name)
    if t.dim() != 4:
        raise ValueError(f"{name} must be 4-D [B,C,H,W], got {tuple(t.shape)}")
    b, c, h, w = t.shape
    st = t.stride()
    if (st[3] != 1 and w > 1) or (st[2] != w and h > 1) or (st[1] != h * w and c > 1):
        raise ValueError(f"{name}: per-image block must be contiguous (strides {st} for shape {tuple(t.shape)})")
    bs = st[0] if b > 1 else c * h * w
    return t.data_ptr(), int(bs)


def _vec(t: Optional[torch.Tensor], n: int, name: str):
    if t is None:
        return None
    _check_f32_cuda(t, name)
    if t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous tensor of {n} elements")
    return t.data_ptr()


def maxpool_out_dim(n: int, kernel: int, stride: int, padding: Optional[int] = None) -> int:
    if padding is None:
        padding = max(0, kernel - 1)
    return capi.lib().pxe_maxpool_out_dim(n, kernel, stride, padding)


def conv_epilogue(x: torch.Tensor, *, y: Optional[torch.Tensor] = None, y2: Optional[torch.Tensor] = None,
                  gamma=None, beta=None, mean=None, var=None, bias=None, act="linear", eps: float = 1e-5,
                  eps_mode: int = capi.EPS_CUDNN, yolo_classes: int = 0,
                  residual: Optional[torch.Tensor] = None, res_alpha: float = 1.0, res_beta: float = 1.0,
                  res_act="linear", pool: Optional[Sequence[int]] = None,
                  y_pool: Optional[torch.Tensor] = None, in_place: bool = True, pool_variant: int = 0,
                  a: Optional[torch.Tensor] = None, b: Optional[torch.Tensor] = None):
    """Fused BN / bias / activation (+ residual, + 2x2 pool, + concat-slot stores).

    Returns ``y`` (or ``(y, y_pool)`` when pooling).  With ``y=None`` the result overwrites ``x``
    (``in_place=True``) or goes to a new tensor; ``y=False`` with pooling skips the
    full-resolution output altogether.  ``a``, ``b``: the layer's coefficients folded once by ``fold_bn`` (then
    gamma / beta / mean / var / bias are not needed); same results, no per-block coefficient table.
    """
    xp, xbs = _slot(x, "x")
    B, Cc, H, W = x.shape
    d = capi.EpilogueDesc()
    d.x, d.x_batch_stride = xp, xbs
    want_full = y is not False
    if y is None:
        y = x if in_place else torch.empty((B, Cc, H, W), device=x.device, dtype=torch.float32)
    if want_full:
        yp, ybs = _slot(y, "y")
        if tuple(y.shape) != (B, Cc, H, W):
            raise ValueError("y shape mismatch")
        d.y, d.y_batch_stride = yp, ybs
    else:
        y = None
    if y2 is not None:
        if tuple(y2.shape) != (B, Cc, H, W):
            raise ValueError("y2 shape mismatch")
        d.y2, d.y2_batch_stride = _slot(y2, "y2")
    d.batch, d.channels, d.height, d.width = B, Cc, H, W
    if gamma is not None:
        d.gamma, d.beta = _vec(gamma, Cc, "gamma"), _vec(beta, Cc, "beta")
        d.mean, d.var = _vec(mean, Cc, "mean"), _vec(var, Cc, "var")
    d.eps, d.eps_mode = eps, eps_mode
    d.bias = _vec(bias, Cc, "bias")
    if a is not None or b is not None:            # coefficients folded once per layer (fold_bn): no per-block table
        d.folded_a, d.folded_b = _vec(a, Cc, "a"), _vec(b, Cc, "b")
    d.act, d.yolo_classes = _act(act), yolo_classes
    if residual is not None:
        if tuple(residual.shape) != (B, Cc, H, W):
            raise ValueError("residual shape mismatch")
        d.residual, d.residual_batch_stride = _slot(residual, "residual")
        d.res_alpha, d.res_beta, d.res_act = res_alpha, res_beta, _act(res_act)
    if pool is not None:
        k, s, pad = pool
        d.pool_kernel, d.pool_stride, d.pool_padding = k, s, pad
        oh, ow = maxpool_out_dim(H, k, s, pad), maxpool_out_dim(W, k, s, pad)
        if y_pool is None:
            y_pool = torch.empty((B, Cc, oh, ow), device=x.device, dtype=torch.float32)
        if tuple(y_pool.shape) != (B, Cc, oh, ow):
            raise ValueError(f"y_pool must be {(B, Cc, oh, ow)}, got {tuple(y_pool.shape)}")
        d.y_pool, d.y_pool_batch_stride = _slot(y_pool, "y_pool")
        d.pool_variant = pool_variant        # capi.POOL_GENERAL: the general pooled kernel whatever the shape (tests)
    capi.check(capi.lib().pxe_conv_epilogue(_stream(), C.byref(d)))
    return (y, y_pool) if pool is not None else y


def activate(kind, x: torch.Tensor) -> torch.Tensor:
    """In-place activation of a contiguous tensor: px::activate (src/Activation.cu:126-133)."""
    _check_f32_cuda(x, "x")
    if not x.is_contiguous():
        raise ValueError("x must be contiguous")
    capi.check(capi.lib().pxe_activate(_stream(), _act(kind), x.data_ptr(), x.numel()))
    return x


def add_bias(out: torch.Tensor, bias: torch.Tensor) -> torch.Tensor:
    """out[b, j, ...] += bias[j] in place: px::addBiasGpu (src/BiasKernels.cu:86-93)."""
    _check_f32_cuda(out, "out")
    if not out.is_contiguous():
        raise ValueError("out must be contiguous")
    B, n = out.shape[0], out.shape[1]
    size = out.numel() // (B * n)
    capi.check(capi.lib().pxe_add_bias(_stream(), out.data_ptr(), _vec(bias, n, "bias"), B, n, size))
    return out


def maxpool(x: torch.Tensor, kernel: int, stride: int, padding: Optional[int] = None,
            out: Optional[torch.Tensor] = None, with_indexes: bool = False):
    """MaxPoolLayer forward.  Returns ``out`` or ``(out, indexes)``."""
    if padding is None:
        padding = max(0, kernel - 1)                       # include/MaxPoolLayer.h:56
    xp, xbs = _slot(x, "x")
    B, Cc, H, W = x.shape
    oh, ow = maxpool_out_dim(H, kernel, stride, padding), maxpool_out_dim(W, kernel, stride, padding)
    if oh <= 0 or ow <= 0:
        raise PxeError(capi.PXE_ERR_BAD_ARG, f"maxpool: empty output {oh}x{ow}")
    if out is None:
        out = torch.empty((B, Cc, oh, ow), device=x.device, dtype=torch.float32)
    if tuple(out.shape) != (B, Cc, oh, ow):
        raise ValueError(f"out must be {(B, Cc, oh, ow)}")
    yp, ybs = _slot(out, "out")
    idx = torch.empty((B, Cc, oh, ow), device=x.device, dtype=torch.int32) if with_indexes else None
    if with_indexes and xbs != Cc * H * W:
        raise ValueError("indexes need a densely packed input")
    capi.check(capi.lib().pxe_maxpool(_stream(), xp, xbs, yp, ybs, idx.data_ptr() if idx is not None else None,
                                      B, Cc, H, W, kernel, stride, padding))
    return (out, idx) if with_indexes else out


def spp(x: torch.Tensor, kernels: Sequence[int], outs: Sequence[torch.Tensor], *, a: Optional[torch.Tensor] = None,
        b: Optional[torch.Tensor] = None, act=None, y_identity: Optional[torch.Tensor] = None) -> Sequence[torch.Tensor]:
    """Stride-1 max pools of one input (default padding kernel-1), one output per kernel size.  With ``act``
    (and optionally the folded coefficients ``a``, ``b`` of fold_bn) ``x`` is a raw convolution output: the
    epilogue is applied as the planes are read, its result goes to ``y_identity`` and into every pool."""
    xp, xbs = _slot(x, "x")
    B, Cc, H, W = x.shape
    n = len(kernels)
    if len(outs) != n:
        raise ValueError("one output per kernel size")
    ptrs, strides = (C.c_void_p * n)(), (C.c_longlong * n)()
    for i, o in enumerate(outs):
        if tuple(o.shape) != (B, Cc, H, W):
            raise ValueError("spp outputs have the input's shape")
        ptrs[i], strides[i] = _slot(o, f"outs[{i}]")
    ks = (C.c_int * n)(*[int(k) for k in kernels])
    if act is None and a is None and y_identity is None:
        capi.check(capi.lib().pxe_spp(_stream(), xp, xbs, B, Cc, H, W, n, ks, ptrs, strides))
        return outs
    if y_identity is not None and tuple(y_identity.shape) != (B, Cc, H, W):
        raise ValueError("y_identity has the input's shape")
    ip, ibs = _slot(y_identity, "y_identity") if y_identity is not None else (None, 0)
    capi.check(capi.lib().pxe_spp_epilogue(_stream(), xp, xbs, B, Cc, H, W, _vec(a, Cc, "a"), _vec(b, Cc, "b"),
                                           _act(act if act is not None else "linear"), ip, ibs, n, ks, ptrs, strides))
    return outs


def upsample(x: torch.Tensor, stride: int = 2, scale: float = 1.0, out: Optional[torch.Tensor] = None):
    xp, xbs = _slot(x, "x")
    B, Cc, H, W = x.shape
    if out is None:
        out = torch.empty((B, Cc, H * stride, W * stride), device=x.device, dtype=torch.float32)
    if tuple(out.shape) != (B, Cc, H * stride, W * stride):
        raise ValueError("out shape mismatch")
    yp, ybs = _slot(out, "out")
    capi.check(capi.lib().pxe_upsample(_stream(), xp, xbs, yp, ybs, B, Cc, H, W, stride, scale))
    return out


def shortcut(x: torch.Tensor, frm: torch.Tensor, alpha: float = 1.0, beta: float = 1.0, act="linear",
             out: Optional[torch.Tensor] = None, out2: Optional[torch.Tensor] = None):
    """out = act(alpha*x + beta*from) for equal shapes (ShortcutLayer forward)."""
    xp, xbs = _slot(x, "x")
    fp, fbs = _slot(frm, "from")
    B, Cc, H, W = x.shape
    if tuple(frm.shape) != (B, Cc, H, W):
        raise ValueError("from shape mismatch")
    if out is None:
        out = torch.empty((B, Cc, H, W), device=x.device, dtype=torch.float32)
    yp, ybs = _slot(out, "out")
    y2p, y2bs = _slot(out2, "out2")
    capi.check(capi.lib().pxe_shortcut(_stream(), xp, xbs, fp, fbs, yp, ybs, y2p, y2bs, B, Cc, H, W,
                                       alpha, beta, _act(act)))
    return out


def shortcut_general(batch, w1, h1, c1, add: torch.Tensor, w2, h2, c2, s1, s2, out: torch.Tensor):
    """px::shortcutGpu for unequal shapes: out = s1*out + s2*add, in place."""
    _check_f32_cuda(add, "add")
    _check_f32_cuda(out, "out")
    capi.check(capi.lib().pxe_shortcut_general(_stream(), batch, w1, h1, c1, add.data_ptr(), w2, h2, c2,
                                               s1, s2, out.data_ptr()))
    return out


def concat(srcs: Sequence[torch.Tensor], out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """RouteLayer forward as one launch."""
    n = len(srcs)
    B, _, H, W = srcs[0].shape
    ch = [int(s.shape[1]) for s in srcs]
    if out is None:
        out = torch.empty((B, sum(ch), H, W), device=srcs[0].device, dtype=torch.float32)
    ptrs, strides = (C.c_void_p * n)(), (C.c_longlong * n)()
    for i, s in enumerate(srcs):
        if s.shape[0] != B or s.shape[2] != H or s.shape[3] != W:
            raise ValueError("route sources must share batch and spatial size")
        ptrs[i], strides[i] = _slot(s, f"srcs[{i}]")
    yp, ybs = _slot(out, "out")
    capi.check(capi.lib().pxe_concat(_stream(), n, ptrs, strides, (C.c_int * n)(*ch), yp, ybs, B, H, W))
    return out


def yolo_activate(x: torch.Tensor, masks: int, classes: int, out: Optional[torch.Tensor] = None):
    _check_f32_cuda(x, "x")
    if not x.is_contiguous():
        raise ValueError("x must be contiguous")
    B = x.shape[0]
    area = x.shape[2] * x.shape[3]
    if out is None:
        out = torch.empty_like(x)
    capi.check(capi.lib().pxe_yolo_activate(_stream(), x.data_ptr(), out.data_ptr(), B, masks, classes, area))
    return out


class DetectionBuffer:
    """Device buffer of detections plus the device-side running count the YOLO decode appends to."""

    def __init__(self, capacity: int, device):
        self.capacity = int(capacity)
        self.dets = torch.empty((self.capacity, 8), device=device, dtype=torch.int32)   # 32-byte records
        self.count = torch.zeros(1, device=device, dtype=torch.int64)
        self._workspace = None

    def reset(self):
        self.count.zero_()

    def workspace(self, nbytes: int) -> torch.Tensor:
        if self._workspace is None or self._workspace.numel() < nbytes:
            self._workspace = torch.empty(max(nbytes, 256), device=self.dets.device, dtype=torch.uint8)
        return self._workspace

    def to_host(self):
        """(structured numpy array of the stored records, total count incl. dropped ones)."""
        total = int(self.count.item())
        n = min(total, self.capacity)
        host = self.dets[:n].cpu().numpy().view(DET_DTYPE).reshape(-1)
        return host, total


def yolo_decode(head: torch.Tensor, mask, anchors, classes: int, net_w: int, net_h: int, threshold: float,
                buf: DetectionBuffer, *, img_w: int = 0, img_h: int = 0, raw: bool = False,
                bias: Optional[torch.Tensor] = None, batch_id_offset: int = 0) -> None:
    """Appends one head's detections to ``buf`` in the reference's emission order.  ``head`` is [B, C, H, W], dense
    NCHW (or a channel slot of a wider NCHW buffer) or dense channels-last; the latter is read where it lies."""
    B, Cc, H, W = head.shape
    d = capi.YoloDecodeDesc()
    nhwc = (not head.is_contiguous()) and head.is_contiguous(memory_format=torch.channels_last) and Cc > 1 and H * W > 1
    if nhwc:
        _check_f32_cuda(head, "head")
        hp, hbs = head.data_ptr(), Cc * H * W
        d.head_channels_last = 1
    else:
        hp, hbs = _slot(head, "head")
    d.head, d.head_batch_stride = hp, hbs
    d.head_is_raw = int(raw)
    d.bias = _vec(bias, Cc, "bias")
    d.batch, d.height, d.width, d.classes = B, H, W, classes
    d.n_masks = len(mask)
    for i, m in enumerate(mask):
        d.mask[i] = int(m)
    d.n_anchor_values = len(anchors)
    for i, a in enumerate(anchors):
        d.anchors[i] = int(a)
    d.net_width, d.net_height = net_w, net_h
    d.image_width, d.image_height = img_w, img_h
    d.threshold, d.batch_id_offset = threshold, batch_id_offset
    if Cc != len(mask) * (classes + 5):
        raise ValueError("head channels must equal masks*(classes+5)")
    need = capi.lib().pxe_yolo_decode_fast_workspace_bytes(B, H, W)
    ws = buf.workspace(need)
    capi.check(capi.lib().pxe_yolo_decode(_stream(), C.byref(d), buf.dets.data_ptr(), buf.capacity,
                                          buf.count.data_ptr(), ws.data_ptr(), ws.numel()))


def centernet_activate(x: torch.Tensor, classes: int, heatmap_bias: float, out: Optional[torch.Tensor] = None):
    _check_f32_cuda(x, "x")
    if not x.is_contiguous():
        raise ValueError("x must be contiguous")
    B = x.shape[0]
    area = x.shape[2] * x.shape[3]
    if out is None:
        out = torch.empty_like(x)
    capi.check(capi.lib().pxe_centernet_activate(_stream(), x.data_ptr(), out.data_ptr(), B, classes, area,
                                                 heatmap_bias))
    return out


def centernet_decode(heat: torch.Tensor, size: torch.Tensor, offset: torch.Tensor, threshold: float,
                     max_detections: int = 100, *, logits: bool = False, heatmap_bias: float = 0.0,
                     img_w: int = 0, img_h: int = 0, batch_id_offset: int = 0, workspace=None,
                     candidate_capacity: int = 0):
    """Returns (dets [B, K, 8] int32 view of 32-byte records, counts [B] int32), both on the device.
    ``candidate_capacity``: see pxe_centernet_decode_desc (0 = default)."""
    hp, hbs = _slot(heat, "heat")
    sp, sbs = _slot(size, "size")
    op, obs = _slot(offset, "offset")
    B, classes, H, W = heat.shape
    d = capi.CenterNetDecodeDesc()
    d.heat, d.heat_batch_stride = hp, hbs
    d.size, d.size_batch_stride = sp, sbs
    d.offset, d.offset_batch_stride = op, obs
    d.heat_is_logit, d.heatmap_bias = int(logits), heatmap_bias
    d.batch, d.classes, d.height, d.width = B, classes, H, W
    d.image_width, d.image_height = img_w, img_h
    d.threshold, d.max_detections, d.batch_id_offset = threshold, max_detections, batch_id_offset
    d.candidate_capacity = candidate_capacity
    need = capi.lib().pxe_centernet_decode_workspace_bytes(B, classes, H, W, max_detections)
    if workspace is None or workspace.numel() < need:
        workspace = torch.empty(max(need, 256), device=heat.device, dtype=torch.uint8)
    dets = torch.empty((B, max_detections, 8), device=heat.device, dtype=torch.int32)
    counts = torch.empty(B, device=heat.device, dtype=torch.int32)
    capi.check(capi.lib().pxe_centernet_decode(_stream(), C.byref(d), dets.data_ptr(), counts.data_ptr(),
                                               workspace.data_ptr(), workspace.numel()))
    return dets, counts


def centernet_to_host(dets: torch.Tensor, counts: torch.Tensor):
    """List of per-image structured arrays."""
    h = dets.cpu().numpy()
    c = counts.cpu().numpy()
    return [h[b, :c[b]].copy().view(DET_DTYPE).reshape(-1) for b in range(h.shape[0])]


def softmax(x: torch.Tensor, groups: int = 1, temperature: float = 1.0, out: Optional[torch.Tensor] = None):
    _check_f32_cuda(x, "x")
    if not x.is_contiguous():
        raise ValueError("x must be contiguous")
    B = x.shape[0]
    inputs = x.numel() // B
    if out is None:
        out = torch.empty_like(x)
    capi.check(capi.lib().pxe_softmax(_stream(), x.data_ptr(), out.data_ptr(), B, inputs, groups, temperature))
    return out


def region_forward(x: torch.Tensor, num: int, coords: int, classes: int, use_softmax: bool = True):
    _check_f32_cuda(x, "x")
    if not x.is_contiguous():
        raise ValueError("x must be contiguous")
    B, _, H, W = x.shape
    out = torch.empty_like(x)
    capi.check(capi.lib().pxe_region_forward(_stream(), x.data_ptr(), out.data_ptr(), B, W, H, num, coords,
                                             classes, int(use_softmax)))
    return out


def nms(dets: np.ndarray, threshold: float) -> np.ndarray:
    """px::nms on host records (structured array of DET_DTYPE)."""
    dets = np.ascontiguousarray(dets, DET_DTYPE)
    out = np.zeros(len(dets), DET_DTYPE)
    n = capi.lib().pxe_nms_host(dets.ctypes.data, len(dets), threshold, out.ctypes.data)
    if n < 0:
        raise PxeError(-n, "pxe_nms_host failed")
    return out[:n].copy()


def nms_device(dets: torch.Tensor, n: int, threshold: float, out: Optional[torch.Tensor] = None,
               workspace: Optional[torch.Tensor] = None):
    """px::nms on the device.  ``dets``: int32 tensor [capacity, 8] of 32-byte records (a DetectionBuffer's
    ``dets``), of which the first ``n`` are valid.  Returns (out [n, 8] int32, count [1] int64), both on the
    device; the first ``count`` records of ``out`` are the survivors in the reference's order."""
    if dets.dtype != torch.int32 or dets.dim() != 2 or dets.shape[1] != 8 or not dets.is_cuda or not dets.is_contiguous():
        raise ValueError("dets must be a contiguous int32 CUDA tensor of shape [capacity, 8]")
    _check_device(dets.device.index, "dets")
    n = int(n)
    if n < 0 or n > dets.shape[0]:
        raise ValueError(f"n = {n} outside 0..{dets.shape[0]}")
    if out is None:
        out = torch.empty((max(n, 1), 8), device=dets.device, dtype=torch.int32)
    count = torch.zeros(1, device=dets.device, dtype=torch.int64)
    need = capi.lib().pxe_nms_workspace_bytes(n)
    if workspace is None or workspace.numel() < need:
        workspace = torch.empty(max(need, 256), device=dets.device, dtype=torch.uint8)
    capi.check(capi.lib().pxe_nms(_stream(), dets.data_ptr(), n, float(threshold), out.data_ptr(), count.data_ptr(),
                                  workspace.data_ptr(), workspace.numel()))
    return out, count


def avgpool(x: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Global average pool: [B, C, H, W] -> [B, C, 1, 1]."""
    xp, xbs = _slot(x, "x")
    B, Cc, H, W = x.shape
    if out is None:
        out = torch.empty((B, Cc, 1, 1), device=x.device, dtype=torch.float32)
    capi.check(capi.lib().pxe_avgpool(_stream(), xp, xbs, out.data_ptr(), out.stride(0), B, Cc, H, W))
    return out


def detect_decode(pred: torch.Tensor, side: int, num: int, classes: int, threshold: float, buf: DetectionBuffer, *,
                  coords: int = 4, squared: bool = False, width: float = 1.0, height: float = 1.0,
                  batch_id_offset: int = 0) -> None:
    """Appends a YOLOv1 detection head's boxes to ``buf``.  ``pred``: [B, side*side*(classes + num*(1+coords))]
    (any trailing shape of that many values per image), contiguous."""
    _check_f32_cuda(pred, "pred")
    if not pred.is_contiguous():
        raise ValueError("pred must be contiguous")
    B = pred.shape[0]
    per = pred.numel() // B
    if per != side * side * (classes + num * (1 + coords)):
        raise ValueError(f"pred has {per} values per image, expected {side * side * (classes + num * (1 + coords))}")
    capi.check(capi.lib().pxe_detect_decode(_stream(), pred.data_ptr(), per, B, side, num, classes, coords, int(squared),
                                            float(width), float(height), float(threshold), buf.dets.data_ptr(),
                                            buf.capacity, buf.count.data_ptr(), batch_id_offset))


# ------------------------------------------------------------------------------ backward-side kernels
def activation_gradient(kind, x: torch.Tensor, delta: torch.Tensor) -> torch.Tensor:
    """delta *= f'(x) in place: px::gradient (src/Activation.cu:135-143)."""
    _check_f32_cuda(x, "x")
    _check_f32_cuda(delta, "delta")
    if not (x.is_contiguous() and delta.is_contiguous()) or x.numel() != delta.numel():
        raise ValueError("x and delta must be contiguous tensors of the same size")
    capi.check(capi.lib().pxe_activation_gradient(_stream(), _act(kind), x.data_ptr(), x.numel(), delta.data_ptr()))
    return delta


def backward_bias(bias_updates: torch.Tensor, delta: torch.Tensor) -> torch.Tensor:
    """bias_updates[f] += sum of delta[:, f] in place: px::backwardBiasGpu (src/BiasKernels.cu:95-111)."""
    _check_f32_cuda(delta, "delta")
    if not delta.is_contiguous():
        raise ValueError("delta must be contiguous")
    B, n = delta.shape[0], delta.shape[1]
    capi.check(capi.lib().pxe_backward_bias(_stream(), _vec(bias_updates, n, "bias_updates"), delta.data_ptr(), B, n,
                                            delta.numel() // (B * n)))
    return bias_updates


def maxpool_backward(delta: torch.Tensor, indexes: torch.Tensor, grad: torch.Tensor) -> torch.Tensor:
    """grad[indexes[i]] += delta[i] in place: px::maxPoolBackwardGpu (src/MaxPoolKernels.cu:61-65)."""
    _check_f32_cuda(delta, "delta")
    _check_f32_cuda(grad, "grad")
    if indexes.dtype != torch.int32 or not indexes.is_cuda or indexes.numel() != delta.numel():
        raise ValueError("indexes must be an int32 CUDA tensor with delta's element count")
    if not (delta.is_contiguous() and indexes.is_contiguous() and grad.is_contiguous()):
        raise ValueError("delta, indexes and grad must be contiguous")
    capi.check(capi.lib().pxe_maxpool_backward(_stream(), delta.data_ptr(), indexes.data_ptr(), grad.data_ptr(), delta.numel()))
    return grad


def upsample_backward(acc: torch.Tensor, out: torch.Tensor, stride: int, scale: float = 1.0) -> torch.Tensor:
    """acc += scale * (sum of the stride x stride block of out above each element): px::upsampleGpu, forward == 0."""
    _check_f32_cuda(acc, "acc")
    _check_f32_cuda(out, "out")
    B, Cc, H, W = acc.shape
    if tuple(out.shape) != (B, Cc, H * stride, W * stride) or not (acc.is_contiguous() and out.is_contiguous()):
        raise ValueError("out must be the contiguous [B, C, H*stride, W*stride] tensor for a contiguous acc [B, C, H, W]")
    capi.check(capi.lib().pxe_upsample_backward(_stream(), acc.data_ptr(), out.data_ptr(), B, Cc, H, W, stride, scale))
    return acc


def constrain(x: torch.Tensor, alpha: float) -> torch.Tensor:
    """x = clamp(x, -alpha, alpha) in place: px::constrainGpu (src/CudaUtils.cu:131-138)."""
    _check_f32_cuda(x, "x")
    if not x.is_contiguous():
        raise ValueError("x must be contiguous")
    capi.check(capi.lib().pxe_constrain(_stream(), x.data_ptr(), x.numel(), alpha))
    return x


def mul(x: torch.Tensor, y: torch.Tensor) -> torch.Tensor:
    """y = x * y in place: px::mulGpu (src/CudaUtils.cu:140-146)."""
    _check_f32_cuda(x, "x")
    _check_f32_cuda(y, "y")
    if not (x.is_contiguous() and y.is_contiguous()) or x.numel() != y.numel():
        raise ValueError("x and y must be contiguous tensors of the same size")
    capi.check(capi.lib().pxe_mul(_stream(), x.data_ptr(), y.data_ptr(), x.numel()))
    return y


def random_uniform(out: torch.Tensor, a: float = 0.0, b: float = 1.0) -> torch.Tensor:
    """px::randomGpu (src/CudaUtils.cu:77-86)."""
    _check_f32_cuda(out, "out")
    capi.check(capi.lib().pxe_random_uniform(_stream(), out.data_ptr(), out.numel(), a, b))
    return out


def random_normal(out: torch.Tensor, mean: float = 0.0, stddev: float = 1.0) -> torch.Tensor:
    """px::randomNormalGpu (src/CudaUtils.cu:110-120)."""
    _check_f32_cuda(out, "out")
    capi.check(capi.lib().pxe_random_normal(_stream(), out.data_ptr(), out.numel(), mean, stddev))
    return out


def yolo_loss(output: torch.Tensor, delta: torch.Tensor, truths: torch.Tensor, truth_counts: torch.Tensor,
              assigned_classes: torch.Tensor, assigned_anchors: torch.Tensor, assigned_boxes: torch.Tensor,
              masks: torch.Tensor, anchors: torch.Tensor, stats: torch.Tensor, cost: torch.Tensor, net_w: int, net_h: int,
              ignore_thr: float = 0.5, truth_thr: float = 1.0, coord_scale: float = 1.0, object_scale: float = 1.0,
              no_object_scale: float = 1.0, class_scale: float = 1.0) -> None:
    """px::yoloLossGpu as one launch; delta, stats (12 floats) and cost (1 float) are updated in place."""
    _check_f32_cuda(output, "output")
    _check_f32_cuda(delta, "delta")
    B, ch, H, W = output.shape
    d = capi.YoloLossDesc()
    d.output, d.delta, d.truths, d.truth_counts = output.data_ptr(), delta.data_ptr(), truths.data_ptr(), truth_counts.data_ptr()
    d.max_truth = truths.shape[1]
    d.assigned_classes, d.assigned_anchors = assigned_classes.data_ptr(), assigned_anchors.data_ptr()
    d.assigned_boxes, d.masks, d.anchors = assigned_boxes.data_ptr(), masks.data_ptr(), anchors.data_ptr()
    d.stats, d.cost = stats.data_ptr(), cost.data_ptr()
    d.batch, d.mask_count, d.classes, d.width, d.height = B, masks.numel(), ch // masks.numel() - 5, W, H
    d.network_width, d.network_height = net_w, net_h
    d.ignore_threshold, d.truth_threshold, d.coord_scale = ignore_thr, truth_thr, coord_scale
    d.object_scale, d.no_object_scale, d.class_scale = object_scale, no_object_scale, class_scale
    capi.check(capi.lib().pxe_yolo_loss(_stream(), C.byref(d)))


def centernet_loss(output: torch.Tensor, delta: torch.Tensor, target_heat: torch.Tensor, target_size: torch.Tensor,
                   target_offset: torch.Tensor, target_mask: torch.Tensor, costs: torch.Tensor, normalizer: float,
                   alpha: float = 2.0, beta: float = 4.0, size_weight: float = 0.1) -> None:
    """px::centerNetLossGpu; delta and costs (3 floats) are updated in place."""
    _check_f32_cuda(output, "output")
    _check_f32_cuda(delta, "delta")
    B, ch, H, W = output.shape
    capi.check(capi.lib().pxe_centernet_loss(_stream(), output.data_ptr(), delta.data_ptr(), target_heat.data_ptr(),
                                             target_size.data_ptr(), target_offset.data_ptr(), target_mask.data_ptr(),
                                             costs.data_ptr(), B, ch - 4, H * W, normalizer, alpha, beta, size_weight))


# ------------------------------------------------------------------------------ channels-last tier
def _nhwc(t: Optional[torch.Tensor], name: str):
    """(pointer, pixel stride) of a logical [B,C,H,W] tensor stored channels-last: a dense channels-last tensor
    or a channel slice of one."""
    if t is None:
        return None, 0
    _check_f32_cuda(t, name)
    if t.dim() != 4:
        raise ValueError(f"{name} must be 4-D [B,C,H,W], got {tuple(t.shape)}")
    b, c, h, w = t.shape
    st = t.stride()
    ps = st[3] if w > 1 else (st[2] // max(w, 1) if h > 1 else (st[0] // max(h * w, 1) if b > 1 else c))
    if ps < c or (c > 1 and st[1] != 1) or (h > 1 and st[2] != w * ps) or (b > 1 and st[0] != h * w * ps):
        raise ValueError(f"{name} is not channels-last (strides {st} for shape {tuple(t.shape)})")
    return t.data_ptr(), int(ps)


def empty_nhwc(shape, device) -> torch.Tensor:
    return torch.empty(tuple(shape), device=device, dtype=torch.float32, memory_format=torch.channels_last)


def fold_bn(channels: int, device, *, gamma=None, beta=None, mean=None, var=None, bias=None, eps: float = 1e-5,
            eps_mode: int = capi.EPS_CUDNN):
    """Folded per-channel coefficients (a, b) of BN inference + bias, computed once per layer."""
    a = torch.empty(channels, device=device, dtype=torch.float32)
    b = torch.empty(channels, device=device, dtype=torch.float32)
    capi.check(capi.lib().pxe_fold_bn(_stream(), _vec(gamma, channels, "gamma"), _vec(beta, channels, "beta"),
                                      _vec(mean, channels, "mean"), _vec(var, channels, "var"),
                                      _vec(bias, channels, "bias"), eps, eps_mode, channels, a.data_ptr(), b.data_ptr()))
    return a, b


def conv_epilogue_nhwc(x: torch.Tensor, *, y: Optional[torch.Tensor] = None, y2: Optional[torch.Tensor] = None,
                       a: Optional[torch.Tensor] = None, b: Optional[torch.Tensor] = None, act="linear",
                       residual: Optional[torch.Tensor] = None, res_alpha: float = 1.0, res_beta: float = 1.0,
                       res_act="linear", pool: Optional[Sequence[int]] = None, y_pool: Optional[torch.Tensor] = None):
    """Fused epilogue on channels-last tensors; ``y=None`` works in place.  With ``pool=(2, 2, padding)`` the
    2x2 max pool is folded in: returns ``(y, y_pool)``, and ``y=False`` skips the full-resolution output."""
    xp, xps = _nhwc(x, "x")
    B, Cc, H, W = x.shape
    want_full = y is not False
    if y is None:
        y = x
    d = capi.EpilogueNhwcDesc()
    d.x, d.x_pixel_stride = xp, xps
    if want_full:
        d.y, d.y_pixel_stride = _nhwc(y, "y")
    else:
        if pool is None:
            raise ValueError("y=False needs pool")
        y = None
    for t, n in ((y, "y"), (y2, "y2"), (residual, "residual")):
        if t is not None and tuple(t.shape) != (B, Cc, H, W):
            raise ValueError(f"{n} has shape {tuple(t.shape)}, expected {(B, Cc, H, W)}")
    if y2 is not None:
        d.y2, d.y2_pixel_stride = _nhwc(y2, "y2")
    if residual is not None:
        d.residual, d.residual_pixel_stride = _nhwc(residual, "residual")
    d.pixels, d.channels = B * H * W, Cc
    d.a, d.b = _vec(a, Cc, "a"), _vec(b, Cc, "b")
    d.act, d.res_alpha, d.res_beta, d.res_act = _act(act), res_alpha, res_beta, _act(res_act)
    if pool is not None:
        k, st, pad = pool
        d.pool_kernel, d.pool_stride, d.pool_padding = k, st, pad
        d.batch, d.height, d.width = B, H, W
        oh, ow = maxpool_out_dim(H, k, st, pad), maxpool_out_dim(W, k, st, pad)
        if y_pool is None:
            y_pool = empty_nhwc((B, Cc, oh, ow), x.device)
        elif tuple(y_pool.shape) != (B, Cc, oh, ow):
            raise ValueError(f"y_pool has shape {tuple(y_pool.shape)}, expected {(B, Cc, oh, ow)}")
        d.y_pool, d.y_pool_pixel_stride = _nhwc(y_pool, "y_pool")
    capi.check(capi.lib().pxe_conv_epilogue_nhwc(_stream(), C.byref(d)))
    return (y, y_pool) if pool is not None else y


def upsample_nhwc(x: torch.Tensor, stride: int, scale: float = 1.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    xp, xps = _nhwc(x, "x")
    B, Cc, H, W = x.shape
    if out is None:
        out = empty_nhwc((B, Cc, H * stride, W * stride), x.device)
    op, ops_ = _nhwc(out, "out")
    capi.check(capi.lib().pxe_upsample_nhwc(_stream(), xp, xps, op, ops_, B, Cc, H, W, stride, scale))
    return out


def maxpool_nhwc(x: torch.Tensor, kernel: int, stride: int, padding: Optional[int] = None,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    xp, xps = _nhwc(x, "x")
    B, Cc, H, W = x.shape
    if padding is None:
        padding = kernel - 1
    oh, ow = maxpool_out_dim(H, kernel, stride, padding), maxpool_out_dim(W, kernel, stride, padding)
    if out is None:
        out = empty_nhwc((B, Cc, oh, ow), x.device)
    op, ops_ = _nhwc(out, "out")
    capi.check(capi.lib().pxe_maxpool_nhwc(_stream(), xp, xps, op, ops_, B, Cc, H, W, kernel, stride, padding))
    return out


def nhwc_to_nchw(x: torch.Tensor) -> torch.Tensor:
    """Dense NCHW copy of a channels-last tensor (for the decoders)."""
    xp, xps = _nhwc(x, "x")
    B, Cc, H, W = x.shape
    out = torch.empty((B, Cc, H, W), device=x.device, dtype=torch.float32)
    capi.check(capi.lib().pxe_nhwc_to_nchw(_stream(), xp, xps, out.data_ptr(), 0, B, Cc, H, W))
    return out


def region_decode(pred: torch.Tensor, width: int, height: int, num: int, coords: int, classes: int, anchors,
                  threshold: float, buf: DetectionBuffer, *, per_image: bool = False, img_w: float = 1.0,
                  img_h: float = 1.0, batch_id_offset: int = 0) -> None:
    """Appends a Region (YOLOv2) head's detections to ``buf``.  ``pred`` is the output of
    :func:`region_forward`.  ``per_image=False`` is the reference's behaviour: every image of the batch decodes
    image 0's predictions (include/RegionLayer.h:363-369)."""
    _check_f32_cuda(pred, "pred")
    if not pred.is_contiguous():
        raise ValueError("pred must be contiguous")
    B = pred.shape[0]
    if pred.numel() != B * width * height * num * (coords + 1 + classes):
        raise ValueError("pred does not have batch * width * height * num * (coords + 1 + classes) values")
    arr = (C.c_float * (2 * num))(*[float(a) for a in list(anchors)[:2 * num]])
    capi.check(capi.lib().pxe_region_decode(_stream(), pred.data_ptr(), B, width, height, num, coords, classes, arr,
                                            int(per_image), float(img_w), float(img_h), float(threshold),
                                            buf.dets.data_ptr(), buf.capacity, buf.count.data_ptr(), batch_id_offset))


def softmax_decode(probs: torch.Tensor, width: float, height: float, threshold: float, buf: DetectionBuffer, *,
                   batch_id_offset: int = 0) -> None:
    """Appends the classifier head's records (SoftmaxLayer::addDetects): one per image whose best class reaches
    the threshold.  ``probs``: [B, classes, ...] contiguous."""
    _check_f32_cuda(probs, "probs")
    if not probs.is_contiguous():
        raise ValueError("probs must be contiguous")
    B = probs.shape[0]
    classes = probs.numel() // B
    capi.check(capi.lib().pxe_softmax_decode(_stream(), probs.data_ptr(), classes, B, classes, float(width), float(height),
                                             float(threshold), buf.dets.data_ptr(), buf.capacity, buf.count.data_ptr(),
                                             batch_id_offset))


def conv_stem(x: torch.Tensor, weights: torch.Tensor, *, a: Optional[torch.Tensor] = None, b: Optional[torch.Tensor] = None,
              act="linear", out: Optional[torch.Tensor] = None, nhwc: bool = False) -> torch.Tensor:
    """First-layer 3x3 / stride 1 / padding 1 convolution fused with its epilogue.  ``x``: NCHW [B, Cin<=4, H, W];
    ``weights``: [Cout, Cin, 3, 3] contiguous; ``a``, ``b``: folded coefficients (:func:`fold_bn`).  The output is
    NCHW, or channels-last with ``nhwc=True``; ``out`` may be a channel slot of a wider buffer of that layout."""
    xp, xbs = _slot(x, "x")
    B, Cin, H, W = x.shape
    _check_f32_cuda(weights, "weights")
    if not weights.is_contiguous() or tuple(weights.shape[1:]) != (Cin, 3, 3):
        raise ValueError(f"weights must be a contiguous [Cout, {Cin}, 3, 3] tensor, got {tuple(weights.shape)}")
    Cout = weights.shape[0]
    if out is None:
        out = empty_nhwc((B, Cout, H, W), x.device) if nhwc else torch.empty((B, Cout, H, W), device=x.device)
    elif tuple(out.shape) != (B, Cout, H, W):
        raise ValueError(f"out has shape {tuple(out.shape)}, expected {(B, Cout, H, W)}")
    d = capi.StemDesc()
    d.x, d.x_batch_stride, d.weights = xp, xbs, weights.data_ptr()
    d.a, d.b = _vec(a, Cout, "a"), _vec(b, Cout, "b")
    d.y, d.y_stride = _nhwc(out, "out") if nhwc else _slot(out, "out")
    d.y_is_nhwc = int(nhwc)
    d.batch, d.in_channels, d.out_channels, d.height, d.width, d.act = B, Cin, Cout, H, W, _act(act)
    capi.check(capi.lib().pxe_conv_stem(_stream(), C.byref(d)))
    return out


def batchnorm_forward_training(x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, *, running_mean=None,
                               running_var=None, exp_avg_factor: float = 0.01, eps: float = 1e-5,
                               eps_mode: int = capi.EPS_CUDNN, act=None, y: Optional[torch.Tensor] = None):
    """Batch normalisation with batch statistics (cudnnBatchNormalizationForwardTraining as the reference's CUDA layers
    call it, include/cuda/ConvLayer.h:285-292; CPU twin src/BatchNorm.cpp:44-60).  Returns ``(y, y_act, save_mean,
    save_scale)``: the normalised tensor, its activation (``None`` without ``act``), the batch mean and
    1 / sqrt(var + eps) (``EPS_CUDNN``) or the population variance (``EPS_CPU``).  The running statistics are updated
    in place."""
    _check_f32_cuda(x, "x")
    if not x.is_contiguous():
        raise ValueError("batchnorm_forward_training: x must be dense NCHW")
    B, Cc, H, W = x.shape
    if y is None:
        y = torch.empty_like(x)
    y_act = torch.empty_like(x) if act is not None else None
    save_mean = torch.empty(Cc, device=x.device, dtype=torch.float32)
    save_scale = torch.empty(Cc, device=x.device, dtype=torch.float32)
    nbytes = capi.lib().pxe_batchnorm_workspace_bytes(B, Cc, H, W)
    ws = torch.empty(nbytes, device=x.device, dtype=torch.uint8)
    d = capi.BnTrainDesc()
    d.x, d.y, d.y_act = x.data_ptr(), y.data_ptr(), (y_act.data_ptr() if y_act is not None else None)
    d.act = _act(act if act is not None else "linear")
    d.batch, d.channels, d.height, d.width = B, Cc, H, W
    d.gamma, d.beta = _vec(gamma, Cc, "gamma"), _vec(beta, Cc, "beta")
    d.running_mean = _vec(running_mean, Cc, "running_mean") if running_mean is not None else None
    d.running_var = _vec(running_var, Cc, "running_var") if running_var is not None else None
    d.exp_avg_factor, d.eps, d.eps_mode = exp_avg_factor, eps, eps_mode
    d.save_mean, d.save_scale = save_mean.data_ptr(), save_scale.data_ptr()
    d.workspace, d.workspace_bytes = ws.data_ptr(), nbytes
    capi.check(capi.lib().pxe_batchnorm_forward_training(_stream(), C.byref(d)))
    return y, y_act, save_mean, save_scale


def batchnorm_backward(x: torch.Tensor, dy: torch.Tensor, gamma: torch.Tensor, save_mean: torch.Tensor,
                       save_scale: torch.Tensor, *, dgamma: Optional[torch.Tensor] = None,
                       dbeta: Optional[torch.Tensor] = None, eps: float = 1e-5, eps_mode: int = capi.EPS_CUDNN,
                       dx: Optional[torch.Tensor] = None) -> torch.Tensor:
    """cudnnBatchNormalizationBackward as the reference's CUDA layers call it (include/cuda/ConvLayer.h:327-332; CPU twin
    src/BatchNorm.cpp:68-98): returns dx; ``dgamma`` and ``dbeta`` are added to."""
    _check_f32_cuda(x, "x")
    _check_f32_cuda(dy, "dy")
    if not (x.is_contiguous() and dy.is_contiguous()) or x.shape != dy.shape:
        raise ValueError("batchnorm_backward: x and dy must be dense NCHW of one shape")
    B, Cc, H, W = x.shape
    if dx is None:
        dx = torch.empty_like(x)
    nbytes = capi.lib().pxe_batchnorm_workspace_bytes(B, Cc, H, W)
    ws = torch.empty(nbytes, device=x.device, dtype=torch.uint8)
    d = capi.BnBackwardDesc()
    d.x, d.dy, d.dx = x.data_ptr(), dy.data_ptr(), dx.data_ptr()
    d.batch, d.channels, d.height, d.width = B, Cc, H, W
    d.gamma = _vec(gamma, Cc, "gamma")
    d.dgamma = _vec(dgamma, Cc, "dgamma") if dgamma is not None else None
    d.dbeta = _vec(dbeta, Cc, "dbeta") if dbeta is not None else None
    d.save_mean, d.save_scale = _vec(save_mean, Cc, "save_mean"), _vec(save_scale, Cc, "save_scale")
    d.eps, d.eps_mode = eps, eps_mode
    d.workspace, d.workspace_bytes = ws.data_ptr(), nbytes
    capi.check(capi.lib().pxe_batchnorm_backward(_stream(), C.byref(d)))
    return dx


def adam_update(x: torch.Tensor, m: torch.Tensor, v: torch.Tensor, beta1: float, beta2: float, rate: float, eps: float,
                t: int) -> torch.Tensor:
    """px::adamGpu (src/Adam.cu:26-47): the parameter step from the moment estimates, in place on ``x``."""
    for name, tns in (("x", x), ("m", m), ("v", v)):
        _check_f32_cuda(tns, name)
        if not tns.is_contiguous() or tns.numel() != x.numel():
            raise ValueError("adam_update: x, m, v must be contiguous and of one size")
    capi.check(capi.lib().pxe_adam_update(_stream(), x.numel(), x.data_ptr(), m.data_ptr(), v.data_ptr(), beta1, beta2, rate, eps, t))
    return x


def softmax_cross_entropy(pred: torch.Tensor, truth: torch.Tensor):
    """px::softmaxCrossEntropy (src/SoftmaxKernel.cu:25-48): returns (delta, error)."""
    _check_f32_cuda(pred, "pred")
    _check_f32_cuda(truth, "truth")
    if not (pred.is_contiguous() and truth.is_contiguous()) or pred.numel() != truth.numel():
        raise ValueError("softmax_cross_entropy: pred and truth must be contiguous and of one size")
    delta, error = torch.empty_like(pred), torch.empty_like(pred)
    capi.check(capi.lib().pxe_softmax_cross_entropy(_stream(), pred.numel(), pred.data_ptr(), truth.data_ptr(), delta.data_ptr(),
                                                    error.data_ptr()))
    return delta, error


# ------------------------------------------------------------------------------ row operators in 32- and 16-bit types
# A call on a token's row is as long as its marshalling: what holds is checked in line, a property at a time, and the
# functions below that word a refusal are called only where something does not.
# The operators are no autograd functions: what they return has no graph, and each gradient is a call of its own.  A graph
# that saved a tensor which a call writes in place finds that out from its version, which the call raises (a replayed
# capture does not).
_DTYPE = {torch.float32: capi.F32, torch.bfloat16: capi.BF16, torch.float16: capi.F16}
_raw_stream = torch._C._cuda_getCurrentRawStream          # of a device's index; what current_stream(...).cuda_stream reads
_current_device = torch._C._cuda_getDevice
_data_ptr = torch.Tensor.data_ptr
_written = torch.autograd.graph.increment_version         # of one tensor or several
_f32 = torch.float32


def _new(shape, dtype, device) -> torch.Tensor:
    """A dense tensor; empty_strided is the cheapest of torch's ways to make one."""
    n = len(shape)
    if n == 1:
        return torch.empty_strided(shape, (1,), dtype=dtype, device=device)
    if n == 2:
        return torch.empty_strided(shape, (shape[1], 1), dtype=dtype, device=device)
    return torch.empty(shape, dtype=dtype, device=device)


def _rows_device(t: torch.Tensor, name: str) -> int:
    """Index of the current device, which a float32, bfloat16 or float16 CUDA tensor has to live on."""
    if not isinstance(t, torch.Tensor) or t.dtype not in _DTYPE or not t.is_cuda:
        raise TypeError(f"{name} must be a float32, bfloat16 or float16 CUDA tensor")
    dev = t.get_device()
    if dev != torch.cuda.current_device():
        _check_device(dev, name)
    return dev


def _like(t: torch.Tensor, shape, dtype, dev: int, name: str) -> torch.Tensor:
    """t, a tensor of this shape and type on device `dev`."""
    if not isinstance(t, torch.Tensor) or t.get_device() < 0:
        raise TypeError(f"{name} must be a CUDA tensor")
    if t.get_device() != dev:
        _check_device(t.get_device(), name)
    if t.shape != shape or t.dtype is not dtype:
        raise ValueError(f"{name} must be {dtype} of shape {tuple(shape)}, got {t.dtype} of {tuple(t.shape)}")
    return t


def _row_stride(t: torch.Tensor, name: str) -> int:
    """Distance in elements between consecutive rows of a [..., n] tensor whose rows are evenly spaced."""
    return t.shape[-1] if t.is_contiguous() else _even_stride(t.shape, t.stride(), name)


def _even_stride(shape, st, name: str) -> int:
    n = shape[-1]
    if n > 1 and st[-1] != 1:
        raise ValueError(f"{name}: rows must be contiguous (strides {st} for shape {tuple(shape)})")
    stride, span = None, 0                    # of the innermost dimension longer than 1; what the dimensions so far cover
    for k in range(len(shape) - 2, -1, -1):
        if shape[k] == 1:
            continue
        if stride is None:
            stride, span = st[k], st[k] * shape[k]
        elif st[k] != span:
            raise ValueError(f"{name}: rows must be evenly spaced (strides {st} for shape {tuple(shape)})")
        else:
            span *= shape[k]
    if stride is None:
        return n
    if stride < n:
        raise ValueError(f"{name}: rows overlap (strides {st} for shape {tuple(shape)})")
    return stride


def _dense_f32(t: Optional[torch.Tensor], n: int, dev: int, name: str):
    """Address of a contiguous float32 tensor of n elements."""
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.dtype is not torch.float32 or t.get_device() != dev:
        _check_f32_cuda(t, name)
    if t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous tensor of {n} elements")
    return t.data_ptr()


def _channels(x: torch.Tensor, name: str, what: str = "channels") -> int:
    shape = x.shape
    if len(shape) == 0 or shape[-1] == 0:
        raise ValueError(f"{name} must have {what}, got shape {tuple(shape)}")
    return shape[-1]


def _norm_weight(weight: Optional[torch.Tensor], channels: int, dtype, dev: int):
    if weight is None:
        return None, capi.F32
    if not isinstance(weight, torch.Tensor) or weight.get_device() != dev:
        _rows_device(weight, "weight")
    if weight.dtype is not torch.float32 and weight.dtype is not dtype:
        raise TypeError(f"weight must be float32 or {dtype}, got {weight.dtype}")
    if weight.dim() != 1 or weight.numel() != channels or not weight.is_contiguous():
        raise ValueError(f"weight must be a contiguous tensor of {channels} elements")
    return weight.data_ptr(), _DTYPE[weight.dtype]


def _rms_norm(x, weight, residual, eps, out, residual_out, e4m3, group):
    shape, dtype, dev = x.shape, x.dtype, x.get_device()
    kind = _DTYPE.get(dtype)
    if kind is None or dev < 0 or dev != _current_device():
        _rows_device(x, "x")
    channels = shape[-1] if shape else 0
    if not channels:
        _channels(x, "x")
    wp, wtype = None, capi.F32
    if weight is not None:
        if weight.dtype is _f32 and weight.dim() == 1 and weight.numel() == channels and weight.get_device() == dev and weight.is_contiguous():
            wp = weight.data_ptr()
        else:
            wp, wtype = _norm_weight(weight, channels, dtype, dev)
    h, rp, rs, hp, hs = x, None, 0, None, 0
    if residual is not None:
        if residual.shape != shape or residual.dtype is not dtype or residual.get_device() != dev:
            _like(residual, shape, dtype, dev, "residual")
        rp, rs = residual.data_ptr(), channels if residual.is_contiguous() else _row_stride(residual, "residual")
        if residual_out is None:
            h, hs = torch.empty_like(x, memory_format=torch.contiguous_format), channels
        else:
            h, hs = _like(residual_out, shape, dtype, dev, "residual_out"), _row_stride(residual_out, "residual_out")
        hp = h.data_ptr()
    elif residual_out is not None:
        raise ValueError("residual_out without a residual")
    device, lead = x.device, shape[:-1]
    rstd = _new(lead, _f32, device)
    y_kind = torch.float8_e4m3fn if e4m3 else dtype
    if out is None:
        y, ys = torch.empty_like(x, dtype=y_kind, memory_format=torch.contiguous_format), channels
    else:
        y, ys = _like(out, shape, y_kind, dev, "out"), _row_stride(out, "out")
    yp, qp, scale, sp, qs = y.data_ptr(), None, None, None, 0
    if e4m3:
        scale = _new(lead + (-(-channels // group) if group else 1,), _f32, device)
        sp, qp, qs, yp, ys = scale.data_ptr(), yp, ys, None, 0
    rows = rstd.numel()
    if rows:
        d = capi.RmsNormDesc(x.data_ptr(), rp, wp, hp, yp, qp, sp, rstd.data_ptr(), channels if x.is_contiguous() else _row_stride(x, "x"),
                             rs, hs, ys, qs, rows, channels, kind, wtype, group, eps)
        rc = capi.lib().pxe_rms_norm(_raw_stream(dev), C.byref(d))
        if rc:
            capi.check(rc)
        if out is not None:
            _written(y)
        if residual_out is not None:
            _written(h)
    return y, scale, h, rstd


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, *, residual: Optional[torch.Tensor] = None,
             eps: float = 1e-6, out: Optional[torch.Tensor] = None, residual_out: Optional[torch.Tensor] = None):
    """Root-mean-square norm over the last dimension, with the residual's addition in front:
    ``h = x + residual``, ``y = h / sqrt(mean(h^2) + eps) * weight``.  Returns ``(y, h, rstd)``; ``h`` is ``x`` itself
    without a residual, ``rstd`` (float32, one for each row) is what :func:`rms_norm_backward` needs.  ``x``: float32,
    bfloat16 or float16 rows, evenly spaced (channels-last pixels: ``x.permute(0, 2, 3, 1)``); ``weight``: float32 or
    x's type.  ``out`` and ``residual_out`` may be ``x`` or ``residual`` (not the same one)."""
    y, _, h, rstd = _rms_norm(x, weight, residual, eps, out, residual_out, False, 0)
    return y, h, rstd


def rms_norm_e4m3(x: torch.Tensor, weight: Optional[torch.Tensor] = None, *, residual: Optional[torch.Tensor] = None,
                  eps: float = 1e-6, group: int = 0, out: Optional[torch.Tensor] = None,
                  residual_out: Optional[torch.Tensor] = None):
    """:func:`rms_norm` with its result in 8 bits for a following product: returns ``(q, scale, h, rstd)`` with ``q``
    float8_e4m3fn and ``y = q * scale``.  ``scale`` is float32 ``[..., ceil(channels / group)]``, one for every ``group``
    (32, 64 or 128) channels of a row, or ``[..., 1]`` for the whole row with ``group=0``."""
    if group not in (0, 32, 64, 128):
        raise ValueError(f"group must be 0, 32, 64 or 128, got {group}")
    return _rms_norm(x, weight, residual, eps, out, residual_out, True, group)


def rms_norm_backward(dy: torch.Tensor, h: torch.Tensor, weight: Optional[torch.Tensor], rstd: torch.Tensor, *,
                      dresidual: Optional[torch.Tensor] = None, dweight: Optional[torch.Tensor] = None,
                      dx: Optional[torch.Tensor] = None):
    """Gradient of :func:`rms_norm`: returns ``(dx, dweight)``.  ``dx`` is the gradient of ``x`` and of the residual
    alike; ``dresidual`` is the gradient that reaches ``h`` past the norm.  ``dweight`` (float32, ``None`` without a
    weight) is added to when given, as :func:`batchnorm_backward` does, and made otherwise.  ``dx`` may be ``dy``,
    ``h`` or ``dresidual``."""
    shape, dtype, dev = dy.shape, dy.dtype, dy.get_device()
    kind = _DTYPE.get(dtype)
    if kind is None or dev < 0 or dev != _current_device():
        _rows_device(dy, "dy")
    channels = shape[-1] if shape else 0
    if not channels:
        _channels(dy, "dy")
    rows = dy.numel() // channels
    if h.shape != shape or h.dtype is not dtype or h.get_device() != dev:
        _like(h, shape, dtype, dev, "h")
    wp, wtype = _norm_weight(weight, channels, dtype, dev)
    rp, rs = None, 0
    if dresidual is not None:
        _like(dresidual, shape, dtype, dev, "dresidual")
        rp, rs = dresidual.data_ptr(), _row_stride(dresidual, "dresidual")
    given_dx = dx
    if dx is None:
        dx, dxs = torch.empty_like(dy, memory_format=torch.contiguous_format), channels
    else:
        dxs = _row_stride(_like(dx, shape, dtype, dev, "dx"), "dx")
    accumulate, ws, wsp, nbytes, dwp = 0, None, None, 0, None
    lib = capi.lib()
    if dweight is not None:
        dwp, accumulate = _dense_f32(dweight, channels, dev, "dweight"), 1
    elif weight is not None:
        dweight = _new((channels,), _f32, dy.device)
        dwp = dweight.data_ptr()
    if dwp is not None:
        nbytes = lib.pxe_rms_norm_backward_workspace_bytes(rows, channels)
        ws = _new((nbytes,), torch.uint8, dy.device)
        wsp = ws.data_ptr()
    d = capi.RmsNormBackwardDesc(dy.data_ptr(), h.data_ptr(), rp, wp, _dense_f32(rstd, rows, dev, "rstd"), dx.data_ptr(), dwp,
                                 _row_stride(dy, "dy"), _row_stride(h, "h"), rs, dxs, rows, channels, kind, wtype, accumulate, wsp, nbytes)
    rc = lib.pxe_rms_norm_backward(_raw_stream(dev), C.byref(d))
    if rc:
        capi.check(rc)
    if given_dx is not None:
        _written(dx)
    if accumulate:
        _written(dweight)
    return dx, dweight


class LogProbs(NamedTuple):
    """What :func:`log_probs` returns; what was not asked for is None."""
    logp: Optional[torch.Tensor]          # [...] float32
    entropy: torch.Tensor                 # [...] float32
    top_logp: Optional[torch.Tensor]      # [..., top] float32, largest first
    top_index: Optional[torch.Tensor]     # [..., top] int32
    stats: torch.Tensor                   # [..., 3] float32, for log_probs_backward


def _grouped_rows(t: torch.Tensor, name: str):
    """(inner, outer stride, row stride) of a [..., n] tensor: evenly spaced rows, or groups of them."""
    shape = t.shape
    if len(shape) > 2 and shape[0] > 1 and t.numel():
        st = t.stride()
        return t.numel() // (shape[0] * shape[-1]), st[0], _even_stride(shape[1:], st[1:], name)
    return 0, 0, _row_stride(t, name)


def _aligned_rows(x: torch.Tensor, inner: int, outer: int, stride: int):
    """A tensor of x's shape and type, its outer and its row stride: dense but for the few elements that put each row at the
    same distance from a 16-byte boundary as x's (its rows as _grouped_rows has them)."""
    shape, vec = x.shape, 16 // x.element_size()
    n, first = shape[-1], x.data_ptr() % 16 // x.element_size()
    stride = n + (stride - n) % vec
    st, at = [1], stride                      # from the innermost dimension out
    for k in range(len(shape) - 2, -1, -1):
        if k == 0 and inner:
            at += (outer - at) % vec
            outer = at
        st.insert(0, at)
        at *= shape[k]
    return torch.empty(first + max(at, n), device=x.device, dtype=x.dtype).as_strided(shape, st, first), outer, stride


def _target(target: torch.Tensor, shape, dev: int):
    if not isinstance(target, torch.Tensor) or target.dtype not in (torch.int64, torch.int32) or not target.is_cuda:
        raise TypeError("target must be an int64 or int32 CUDA tensor")
    if target.get_device() != dev:
        _check_device(target.get_device(), "target")
    if target.shape != shape or not target.is_contiguous():
        raise ValueError(f"target must be a contiguous tensor of shape {tuple(shape)}, got {tuple(target.shape)}")
    return target.data_ptr(), int(target.dtype is torch.int64)


def log_probs(x: torch.Tensor, target: Optional[torch.Tensor] = None, *, top: int = 0, temperature: float = 1.0) -> LogProbs:
    """Log probabilities of given classes, the entropy and the ``top`` (up to 32) most likely classes of every row of
    ``x`` [..., classes] (float32, bfloat16 or float16; a slice such as ``x[:, :-1]`` is read where it lies).  A negative
    ``target`` marks a row that is not used: zeros, and -1 for its alternatives.  Ties go to the lower class."""
    whole, dtype, dev = x.shape, x.dtype, x.get_device()
    kind = _DTYPE.get(dtype)
    if kind is None or dev < 0 or dev != _current_device():
        _rows_device(x, "x")
    classes = whole[-1] if whole else 0
    if not classes:
        _channels(x, "x", "classes")
    if not 0 <= top <= 32 or top > classes:
        raise ValueError(f"top must lie in 0..{min(32, classes)}, got {top}")
    device, shape = x.device, whole[:-1]
    logp = top_logp = top_index = tp = lp = vp = ip = None
    is64 = 0
    if target is not None:
        tp, is64 = _target(target, shape, dev)
        logp = _new(shape, _f32, device)
        lp = logp.data_ptr()
    entropy, stats = _new(shape, _f32, device), _new(shape + (3,), _f32, device)
    if top:
        top_logp, top_index = _new(shape + (top,), _f32, device), _new(shape + (top,), torch.int32, device)
        vp, ip = top_logp.data_ptr(), top_index.data_ptr()
    inner, outer, stride = (0, 0, classes) if x.is_contiguous() else _grouped_rows(x, "x")
    d = capi.LogProbsDesc(x.data_ptr(), tp, lp, entropy.data_ptr(), stats.data_ptr(), vp, ip, entropy.numel(), inner, outer, stride, classes,
                          kind, is64, top, temperature)
    rc = capi.lib().pxe_log_probs(_raw_stream(dev), C.byref(d))
    if rc:
        capi.check(rc)
    return LogProbs(logp, entropy, top_logp, top_index, stats)


def log_probs_backward(x: torch.Tensor, target: Optional[torch.Tensor], stats: torch.Tensor, dlogp: Optional[torch.Tensor] = None, *,
                       dentropy: Optional[torch.Tensor] = None, temperature: float = 1.0,
                       dx: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient of :func:`log_probs` with respect to ``x``, from the gradients of ``logp`` and of ``entropy`` (float32, one
    for each row; either may be missing).  ``stats`` and ``temperature`` are the forward call's.  ``dx`` may be ``x``;
    without it the gradient is dense, but for the few elements that keep its rows at the distances of x's from a 16-byte
    boundary."""
    shape, dtype, dev = x.shape, x.dtype, x.get_device()
    kind = _DTYPE.get(dtype)
    if kind is None or dev < 0 or dev != _current_device():
        _rows_device(x, "x")
    classes = shape[-1] if shape else 0
    if not classes:
        _channels(x, "x", "classes")
    rows = x.numel() // classes
    if dlogp is None and dentropy is None:
        raise ValueError("neither dlogp nor dentropy")
    if dlogp is not None and target is None:
        raise ValueError("dlogp without target")
    tp, is64 = _target(target, shape[:-1], dev) if target is not None else (None, 0)
    given, xp = dx is not None, x.data_ptr()
    if not given:
        if xp % 16 == 0 and x.is_contiguous():
            dx = torch.empty_strided(shape, x.stride(), device=x.device, dtype=dtype)
            inner, outer, stride = 0, 0, classes
            dx_outer, dx_stride = outer, stride
        else:
            inner, outer, stride = _grouped_rows(x, "x")
            dx, dx_outer, dx_stride = _aligned_rows(x, inner, outer, stride)
    else:
        inner, outer, stride = _grouped_rows(x, "x")
        _, dx_outer, dx_stride = _grouped_rows(_like(dx, shape, dtype, dev, "dx"), "dx")
    d = capi.LogProbsBackwardDesc(xp, tp, _dense_f32(stats, 3 * rows, dev, "stats"), _dense_f32(dlogp, rows, dev, "dlogp"),
                                  _dense_f32(dentropy, rows, dev, "dentropy"), dx.data_ptr(), rows, inner, outer, stride, dx_outer,
                                  dx_stride, classes, kind, is64, temperature)
    rc = capi.lib().pxe_log_probs_backward(_raw_stream(dev), C.byref(d))
    if rc:
        capi.check(rc)
    if given:
        _written(dx)
    return dx


class AdamW:
    """An AdamW step over many tensors at once (pxe_adamw_update), with its state.

    ``params``: contiguous CUDA tensors of one type (float32, bfloat16 or float16) on one device.  ``state_bits=32``
    keeps ``m`` and ``v`` as float32; ``state_bits=8`` keeps ``m`` and the root of ``v`` as float8_e4m3fn codes with a
    float32 scale for every 256 elements (``m_scale``, ``v_scale``).  Codes are 6 to 12 % apart: rounded to nearest, as
    they are without a ``seed``, they lose what a step moves by less, and over many steps the moments stop following the
    gradients.  Training takes a ``seed`` (a whole number above 0): codes are then rounded up or down at random, so that
    on average nothing is lost, and the same steps with the same seed give the same bits.  ``master=True`` keeps float32 copies of 16-bit
    parameters and updates those.  All are lists, one tensor for each parameter; lists of an earlier state can be given
    instead (a loaded checkpoint) and are then updated in place.  The plan holds the parameters and the state; a tensor
    of either that was replaced, or whose memory has moved since, is refused by :meth:`step`.  To load another state
    later, copy into the tensors or make a new plan."""

    def __init__(self, params: Sequence[torch.Tensor], *, state_bits: int = 32, m=None, v=None, m_scale=None, v_scale=None, master=None,
                 seed: Optional[int] = None):
        if state_bits not in (32, 8):
            raise ValueError(f"state_bits must be 32 or 8, got {state_bits}")
        if seed is not None and (state_bits != 8 or not 0 < seed < 1 << 64):
            raise ValueError(f"seed must be a whole number from 1 to 2^64 - 1, for states in 8 bits, got {seed} for {state_bits}")
        self.params = list(params)
        self.state_bits = state_bits
        self._dtype, self._device = torch.float32, None
        dev = -1
        if self.params:
            dev = _rows_device(self.params[0], "params[0]")
            self._dtype, self._device = self.params[0].dtype, self.params[0].device
        for i, p in enumerate(self.params):
            if p.dtype is not self._dtype or p.get_device() != dev:
                _rows_device(p, f"params[{i}]")
                raise TypeError(f"params[{i}] is {p.dtype}, the others {self._dtype}: one plan for each type")
            if not p.is_contiguous():
                raise ValueError(f"params[{i}] must be contiguous")
        self._sizes = [p.numel() for p in self.params]
        self._shapes = [p.shape for p in self.params]
        blocks = [-(-n // capi.ADAMW_BLOCK) for n in self._sizes]
        small = state_bits == 8
        if (m is None) != (v is None) or (not small and (m_scale is not None or v_scale is not None)) \
                or (small and not ((m is None) == (m_scale is None) == (v_scale is None))):
            raise ValueError("an earlier state is m and v, and m_scale and v_scale with 8 bits")
        state = torch.float8_e4m3fn if small else torch.float32
        self.m, self.v = (self._state(t, self._sizes, state, n) for t, n in ((m, "m"), (v, "v")))
        self.m_scale, self.v_scale = ((self._state(t, blocks, torch.float32, n) for t, n in ((m_scale, "m_scale"), (v_scale, "v_scale")))
                                      if small else (None, None))
        self.master = None
        if master is not None and master is not False:
            if self._dtype == torch.float32:
                raise ValueError("a master copy of float32 parameters")
            self.master = self._state(None if master is True else master, self._sizes, torch.float32, "master")
            if master is True:
                for w, p in zip(self.master, self.params):
                    w.copy_(p.detach().reshape(-1))
        count = len(self.params)
        # what the table's addresses belong to, kept so that nothing else can take their place, and the addresses
        self._held = [(name, list(tensors), list(map(_data_ptr, tensors))) for name, tensors in
                      (("params", self.params), ("m", self.m), ("v", self.v), ("m_scale", self.m_scale), ("v_scale", self.v_scale),
                       ("master", self.master)) if tensors is not None]
        # the table the call reads, a pxe_adamw_tensor a row; the gradients' addresses change from step to step
        self._table = np.zeros((max(count, 1), C.sizeof(capi.AdamwTensor) // 8), dtype=np.uint64)
        column = lambda name: self._table[:count, getattr(capi.AdamwTensor, name).offset // 8]  # noqa: E731
        column("n")[:] = self._sizes
        for name, _, ptrs in self._held:
            column("param" if name == "params" else name)[:] = ptrs
        self._grads = column("grad")
        d = self._desc = capi.AdamwDesc()
        d.tensors, d.count, d.state_bits, d.param_type = self._table.ctypes.data, count, state_bits, _DTYPE[self._dtype]
        d.seed = seed or 0

    def _state(self, given, sizes, dtype, name):
        if given is None:                    # one buffer, every tensor on a 256-byte boundary
            unit = 256 // dtype.itemsize
            at = [0]
            for n in sizes:
                at.append(at[-1] + -(-n // unit) * unit)
            buf = torch.zeros(at[-1], device=self._device, dtype=torch.float32 if dtype == torch.float32 else torch.uint8).view(dtype)
            return [buf[o:o + n] for o, n in zip(at, sizes)]
        given = list(given)
        if len(given) != len(sizes):
            raise ValueError(f"{name} has {len(given)} tensors for {len(sizes)} parameters")
        dev = self._device.index if sizes else -1
        for i, (t, n) in enumerate(zip(given, sizes)):
            if t.dtype is not dtype or t.numel() != n or t.get_device() != dev or not t.is_contiguous():
                raise ValueError(f"{name}[{i}] must be a contiguous {dtype} tensor of {n} elements on {self._device}")
        return given

    def _scalar(self, t, dtype, name):
        if not t.is_cuda or t.dtype != dtype or t.numel() != 1:
            raise TypeError(f"{name} must be a number or a {dtype} CUDA tensor of one element")
        _check_device(t.device.index, name)
        return t.data_ptr()

    def step(self, grads: Sequence[torch.Tensor], *, rate, t, beta1: float = 0.9, beta2: float = 0.999, eps: float = 1e-8,
             weight_decay: float = 0.0, grad_scale=1.0, skip: Optional[torch.Tensor] = None) -> None:
        """One step, in place on the parameters and the state.  ``grads``: one contiguous tensor for each parameter, all
        of one type (float32 or the parameters' own; any of the three types for float32 parameters).  ``t`` counts steps
        from 1.  ``rate``, ``grad_scale`` (float32) and ``t`` (int64) may be CUDA tensors of one element, which a captured
        step reads at every replay; a ``t`` below 1 there makes the step do nothing, and so does ``skip``, a float32 one,
        when it is not 0."""
        count = len(self._sizes)
        if len(grads) != count:
            raise ValueError(f"{len(grads)} gradients for {count} parameters")
        if count == 0:
            return
        dev = self._device.index
        if dev != torch.cuda.current_device():
            _check_device(dev, "params")
        for name, _, ptrs in self._held:
            if list(map(_data_ptr, getattr(self, name))) != ptrs:
                raise RuntimeError(f"{name}: a tensor was replaced or its memory has moved since this plan was made; make a new one")
        kind = getattr(grads[0], "dtype", None)
        if kind not in _DTYPE:
            raise TypeError(f"gradients must be float32, bfloat16 or float16 tensors, got {kind}")
        ptrs = []
        for i, (g, shape) in enumerate(zip(grads, self._shapes)):
            if not isinstance(g, torch.Tensor):
                raise TypeError(f"grads[{i}] is not a tensor")
            if g.dtype is not kind or g.shape != shape or g.get_device() != dev or not g.is_contiguous():
                raise ValueError(f"gradients must be contiguous {kind} tensors on {self._device} of the parameters' shapes; "
                                 f"got {g.dtype} on {g.device} of shape {tuple(g.shape)} for {tuple(shape)}")
            ptrs.append(g.data_ptr())
        self._grads[:] = ptrs
        d = self._desc
        d.grad_type = _DTYPE[kind]
        d.rate_device = d.t_device = d.grad_scale_device = d.skip_device = None
        if isinstance(rate, torch.Tensor):
            d.rate_device = self._scalar(rate, torch.float32, "rate")
        else:
            d.rate = rate
        if isinstance(t, torch.Tensor):
            d.t_device = self._scalar(t, torch.int64, "t")
        else:
            d.t = t
        if isinstance(grad_scale, torch.Tensor):
            d.grad_scale_device = self._scalar(grad_scale, torch.float32, "grad_scale")
        else:
            d.grad_scale = grad_scale
        if skip is not None:
            d.skip_device = self._scalar(skip, torch.float32, "skip")
        d.beta1, d.beta2, d.eps, d.weight_decay = beta1, beta2, eps, weight_decay
        capi.check(capi.lib().pxe_adamw_update(_raw_stream(dev), C.byref(d)))
        _written(self.params)
