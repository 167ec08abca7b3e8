"""Torch-facing wrappers over the C ABI (include/frcnn_hip.h).

torch is used for device memory and streams only: every wrapper allocates its outputs with
torch.empty on the inputs' device, hands raw device pointers plus the current HIP stream to
libfrcnn_hip.so, and returns without synchronising.  Batched entry points take a leading image
dimension so that a whole batch is one launch (the reference loops over images in Python:
RPN/rpn.py:63,74,80,105; ROIHead/roi_head.py:99,178).

Also exports `nms` and `MultiScaleRoIAlign` with torchvision's signatures, because the reference
imports those two names (RPN/rpn.py:18, ROIHead/roi_head.py:26, ROIHead/roi_pooling.py:18).
"""
import collections
import ctypes
import functools
import os
import math

import numpy as np
import torch

from . import _lib


def _need_gpu(*tensors):
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise _lib.FrcnnError(
                "objectdetection_amd kernels run on a HIP device only (got a %s tensor); "
                "there is no CPU fallback" % t.device)


def _f32c(t):
    if t.dtype != torch.float32:
        t = t.to(torch.float32)
    return t.detach().contiguous()


def _ptr(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else ctypes.c_void_p(0)


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _host_f32(values):
    a = np.ascontiguousarray(np.asarray(values, dtype=np.float32))
    return a, a.ctypes.data_as(ctypes.c_void_p)


# --------------------------------------------------------------------------------- K1 anchors
def base_anchors(sizes, ratios):
    """(size, ratio) per base anchor -> (na,4) CPU fp32 tensor (anchor_generator.py:43-64)."""
    s, sp = _host_f32(sizes)
    r, rp = _host_f32(ratios)
    out = np.empty((len(s), 4), np.float32)
    rc = _lib.load().frcnn_base_anchors_f32(sp, rp, len(s), out.ctypes.data_as(ctypes.c_void_p))
    _lib.check(rc, "base_anchors")
    return torch.from_numpy(out)


def anchor_grid(base, fh, fw, stride_y, stride_x):
    """One level of generate_anchor -> (fh*fw, na, 4) (anchor_generator.py:66-95)."""
    _need_gpu(base)
    base = _f32c(base)
    na = base.shape[0]
    out = torch.empty((fh * fw, na, 4), dtype=torch.float32, device=base.device)
    with torch.cuda.device(base.device):
        rc = _lib.load().frcnn_anchor_grid_f32(_ptr(base), na, fh, fw, float(stride_y), float(stride_x),
                                               _ptr(out), _stream())
    _lib.check(rc, "anchor_grid")
    return out


# --------------------------------------------------------------------------- K2 flatten, top-k
def rpn_flatten(list_cls, list_regs):
    """RPN/rpn.py:56-57: -> scores (B, A), deltas (B, A, 4); flat index = level_off + cell*na + a."""
    _need_gpu(*list_cls, *list_regs)
    B = list_cls[0].shape[0]
    na = list_cls[0].shape[1]
    sizes = [c.shape[2] * c.shape[3] * c.shape[1] for c in list_cls]
    A = sum(sizes)
    dev = list_cls[0].device
    scores = torch.empty((B, A), dtype=torch.float32, device=dev)
    deltas = torch.empty((B, A, 4), dtype=torch.float32, device=dev)
    off = 0
    lib = _lib.load()
    with torch.cuda.device(dev):
        for cls, reg, sz in zip(list_cls, list_regs, sizes):
            if cls.shape[1] != na or reg.shape[1] != 4 * na or reg.shape[2:] != cls.shape[2:]:
                raise ValueError("rpn head outputs disagree: cls %s reg %s" % (tuple(cls.shape), tuple(reg.shape)))
            cls_c, reg_c = _f32c(cls), _f32c(reg)
            rc = lib.frcnn_rpn_flatten_f32(_ptr(cls_c), _ptr(reg_c), B, na, cls.shape[2], cls.shape[3], off, A,
                                           _ptr(scores), _ptr(deltas), _stream())
            _lib.check(rc, "rpn_flatten")
            off += sz
    return scores, deltas


def topk_desc(scores, k, want_values=True, max_slices=0):
    """Per-row sorted top-k (RPN/rpn.py:65-66).  scores (B,n) -> values (B,k), indices (B,k) int32.
    max_slices caps the workgroups a row is split over (0: the library decides, 1: one per row -- for
    callers that run beside a chip-filling kernel, see pipeline.py); results do not depend on it."""
    _need_gpu(scores)
    scores = _f32c(scores)
    B, n = scores.shape
    if k > n:
        raise ValueError("k (%d) > n (%d)" % (k, n))
    dev = scores.device
    vals = torch.empty((B, k), dtype=torch.float32, device=dev) if want_values else None
    idx = torch.empty((B, k), dtype=torch.int32, device=dev)
    lib = _lib.load()
    nbytes = lib.frcnn_topk_workspace_bytes(B, n, k)
    ws = torch.empty((max(nbytes, 16),), dtype=torch.uint8, device=dev)
    with torch.cuda.device(dev):
        rc = lib.frcnn_topk_desc_ex_f32(_ptr(scores), B, n, k, _ptr(vals), _ptr(idx), _ptr(ws), nbytes,
                                        int(max_slices), _stream())
    _lib.check(rc, "topk_desc")
    return vals, idx


def _level_table(tensors, na, per_cell):
    """Host arrays for the C ABI's level tables: device pointers and (h, w) of every level."""
    ts = []
    hw = []
    for t in tensors:
        if t.shape[1] != per_cell * na:
            raise ValueError("rpn head output %s does not have %d channels" % (tuple(t.shape), per_cell * na))
        ts.append(_f32c(t))
        hw += [t.shape[2], t.shape[3]]
    ptrs = (ctypes.c_void_p * len(ts))(*[t.data_ptr() for t in ts])
    hw_arr = (ctypes.c_int32 * len(hw))(*hw)
    return ts, ptrs, hw_arr


def rpn_in_place_supported(list_cls, k, max_slices=0):
    """True where topk_desc_nchw / decode_clip_filter_nchw cover the head outputs (else: rpn_flatten first)."""
    if len(list_cls) > 6:
        return False
    B, na = list_cls[0].shape[0], list_cls[0].shape[1]
    A = sum(c.shape[1] * c.shape[2] * c.shape[3] for c in list_cls)
    return bool(_lib.load().frcnn_topk_desc_nchw_supported(B, A, int(k), int(max_slices)))


def topk_desc_nchw(list_cls, k, want_values=True, max_slices=0):
    """topk_desc over the flattened scores of RPN/rpn.py:56, read from the (B,na,h,w) head outputs in place."""
    _need_gpu(*list_cls)
    B, na = list_cls[0].shape[0], list_cls[0].shape[1]
    ts, ptrs, hw = _level_table(list_cls, na, 1)
    A = na * sum(hw[2 * i] * hw[2 * i + 1] for i in range(len(ts)))
    dev = ts[0].device
    vals = torch.empty((B, k), dtype=torch.float32, device=dev) if want_values else None
    idx = torch.empty((B, k), dtype=torch.int32, device=dev)
    lib = _lib.load()
    nbytes = lib.frcnn_topk_workspace_bytes(B, A, k)
    ws = torch.empty((max(nbytes, 16),), dtype=torch.uint8, device=dev)
    with torch.cuda.device(dev):
        rc = lib.frcnn_topk_desc_nchw_f32(ctypes.cast(ptrs, ctypes.c_void_p), ctypes.cast(hw, ctypes.c_void_p),
                                          len(ts), na, B, k, _ptr(vals), _ptr(idx), _ptr(ws), nbytes, int(max_slices),
                                          _stream())
    _lib.check(rc, "topk_desc_nchw")
    return vals, idx


def decode_clip_filter_nchw(anchors, list_regs, top_idx, top_score, image_h, image_w, min_size):
    """decode_clip_filter with the deltas read from the (B,4na,h,w) head outputs in place."""
    _need_gpu(anchors, top_idx, top_score, *list_regs)
    B = list_regs[0].shape[0]
    na = list_regs[0].shape[1] // 4
    ts, ptrs, hw = _level_table(list_regs, na, 4)
    A = na * sum(hw[2 * i] * hw[2 * i + 1] for i in range(len(ts)))
    anchors, top_score = _f32c(anchors), _f32c(top_score)
    top_idx = top_idx.contiguous()
    if top_idx.dtype != torch.int32:
        top_idx = top_idx.to(torch.int32)
    k = top_idx.shape[1]
    if anchors.dim() == 2:
        stride = 0
        if anchors.shape[0] != A:
            raise ValueError("anchors (%d) and head outputs (%d) disagree" % (anchors.shape[0], A))
    else:
        stride = A * 4
        if anchors.shape[0] != B or anchors.shape[1] != A:
            raise ValueError("anchors %s vs head outputs (B=%d, A=%d)" % (tuple(anchors.shape), B, A))
    dev = ts[0].device
    boxes = torch.empty((B, k, 4), dtype=torch.float32, device=dev)
    scores = torch.empty((B, k), dtype=torch.float32, device=dev)
    src = torch.empty((B, k), dtype=torch.int32, device=dev)
    count = torch.empty((B,), dtype=torch.int32, device=dev)
    with torch.cuda.device(dev):
        rc = _lib.load().frcnn_decode_clip_filter_nchw_f32(
            _ptr(anchors), stride, ctypes.cast(ptrs, ctypes.c_void_p), ctypes.cast(hw, ctypes.c_void_p), len(ts), na,
            _ptr(top_idx), _ptr(top_score), B, k, float(image_h), float(image_w), float(min_size), _ptr(boxes),
            _ptr(scores), _ptr(src), _ptr(count), _stream())
    _lib.check(rc, "decode_clip_filter_nchw")
    return boxes, scores, src, count


def rpn_proposals_nchw(list_cls, list_regs, anchors, k, image_h, image_w, min_size, nms_threshold, max_keep,
                       max_slices=0, rounds=None, workspace=None):
    """RPN/rpn.py:54-85 in one library call (frcnn_rpn_proposals_nchw_f32): topk_desc_nchw -> decode_clip_filter_nchw
    -> nms_sorted -> gather_boxes with their intermediates in one workspace -- same results, a quarter of the host
    work.  -> (props (B,max_keep,4) zero-padded, n_keep (B) int32, workspace) ; pass the returned workspace back in
    to reuse it (it is as large as the sizes need, or a new one is made)."""
    _need_gpu(anchors, *list_cls, *list_regs)
    B, na = list_cls[0].shape[0], list_cls[0].shape[1]
    ts_c, ptrs_c, hw = _level_table(list_cls, na, 1)
    ts_r, ptrs_r, hw_r = _level_table(list_regs, na, 4)
    if list(hw) != list(hw_r):
        raise ValueError("rpn_proposals_nchw: score and delta maps disagree in size")
    A = na * sum(hw[2 * i] * hw[2 * i + 1] for i in range(len(ts_c)))
    anchors = _f32c(anchors)
    if anchors.dim() == 2:
        stride = 0
        if anchors.shape[0] != A:
            raise ValueError("anchors (%d) and head outputs (%d) disagree" % (anchors.shape[0], A))
    else:
        stride = A * 4
        if anchors.shape[0] != B or anchors.shape[1] != A:
            raise ValueError("anchors %s vs head outputs (B=%d, A=%d)" % (tuple(anchors.shape), B, A))
    dev = ts_c[0].device
    k, max_keep = int(k), int(max_keep)
    lib = _lib.load()
    nbytes = lib.frcnn_rpn_proposals_workspace_bytes(B, A, k, max_keep)
    if workspace is None or workspace.numel() < nbytes or workspace.device != dev:
        workspace = torch.empty((max(nbytes, 16),), dtype=torch.uint8, device=dev)
    props = torch.empty((B, max_keep, 4), dtype=torch.float32, device=dev)
    n_keep = torch.empty((B,), dtype=torch.int32, device=dev)
    max_blocks, used = 0, None
    if rounds is not None and lib.frcnn_nms_workspace_bytes(B, k) > 0:
        max_blocks, used = rounds.bound((dev.index, B, k, max_keep, float(nms_threshold)), B)
    with torch.cuda.device(dev):
        rc = lib.frcnn_rpn_proposals_nchw_f32(
            ctypes.cast(ptrs_c, ctypes.c_void_p), ctypes.cast(ptrs_r, ctypes.c_void_p), ctypes.cast(hw, ctypes.c_void_p),
            len(ts_c), na, _ptr(anchors), stride, B, k, float(image_h), float(image_w), float(min_size),
            float(nms_threshold), max_keep, _ptr(props), _ptr(n_keep), _ptr(workspace), workspace.numel(),
            int(max_slices), max_blocks, used.data_ptr() if used is not None else None, _stream())
    _lib.check(rc, "rpn_proposals_nchw")
    return props, n_keep, workspace


# ------------------------------------------------------------------ K3 decode / clip / filter
def box_regression(box, regs):
    _need_gpu(box, regs)
    box, regs = _f32c(box), _f32c(regs)
    n = box.shape[0]
    if box.dim() != 2 or box.shape[1] != 4 or regs.dim() != 2 or regs.shape[0] != n or regs.shape[1] % 4:
        raise ValueError("box_regression expects box (n,4) and regression_params (n,4K); got %s, %s"
                         % (tuple(box.shape), tuple(regs.shape)))
    K = regs.shape[1] // 4
    out = torch.empty_like(regs)
    with torch.cuda.device(box.device):
        rc = _lib.load().frcnn_box_regression_f32(_ptr(box), _ptr(regs), n, K, _ptr(out), _stream())
    _lib.check(rc, "box_regression")
    return out


def box_regression_backward(box, regs, grad_out, want_box_grad=True):
    """-> (grad_regs (n,4K), grad_box (n,4) or None): torch autograd's result through utils.py:173-208."""
    _need_gpu(box, regs, grad_out)
    box, regs, grad_out = _f32c(box), _f32c(regs), _f32c(grad_out)
    n = box.shape[0]
    if regs.shape != grad_out.shape or regs.shape[0] != n or regs.shape[1] % 4:
        raise ValueError("box_regression_backward: shapes %s %s %s" % (tuple(box.shape), tuple(regs.shape),
                                                                        tuple(grad_out.shape)))
    K = regs.shape[1] // 4
    grad_regs = torch.empty_like(regs)
    grad_box = torch.empty_like(box) if want_box_grad else None
    with torch.cuda.device(box.device):
        rc = _lib.load().frcnn_box_regression_backward_f32(_ptr(box), _ptr(regs), _ptr(grad_out), n, K,
                                                           _ptr(grad_regs), _ptr(grad_box) if want_box_grad else None,
                                                           _stream())
    _lib.check(rc, "box_regression_backward")
    return grad_regs, grad_box


class BoxRegression(torch.autograd.Function):
    """Differentiable decode: forward and backward are the HIP kernels."""

    @staticmethod
    def forward(ctx, box, regs):
        ctx.save_for_backward(box, regs)
        return box_regression(box.detach(), regs.detach())

    @staticmethod
    def backward(ctx, grad_out):
        box, regs = ctx.saved_tensors
        need_box = ctx.needs_input_grad[0]
        grad_regs, grad_box = box_regression_backward(box.detach(), regs.detach(), grad_out, need_box)
        return (grad_box if need_box else None), (grad_regs if ctx.needs_input_grad[1] else None)


def resize_pad_into(image, out_h, out_w, canvas):
    """Bilinear resize of image (C,h,w) to (out_h,out_w) into the top-left of canvas (C,H,W), zeros elsewhere
    (generalized_transform.py:58-64 + utils.py:362-369 fused).  canvas is written in full."""
    _need_gpu(image, canvas)
    image = _f32c(image)
    if image.dim() != 3 or canvas.dim() != 3 or canvas.shape[0] != image.shape[0] or not canvas.is_contiguous() \
            or canvas.dtype != torch.float32:
        raise ValueError("resize_pad_into expects image (C,h,w) and a contiguous fp32 canvas (C,H,W)")
    C, h, w = image.shape
    with torch.cuda.device(image.device):
        rc = _lib.load().frcnn_resize_pad_f32(_ptr(image), C, h, w, int(out_h), int(out_w), _ptr(canvas),
                                              canvas.shape[1], canvas.shape[2], _stream())
    _lib.check(rc, "resize_pad")
    return canvas


def resize_pad_batch(images, out_sizes, batch):
    """resize_pad_into for every image of a list in ONE launch: images[i] (C,h_i,w_i) -> batch[i] (C,H,W)."""
    _need_gpu(batch, *images)
    imgs = [_f32c(im) for im in images]
    n = len(imgs)
    if batch.dim() != 4 or batch.shape[0] != n or not batch.is_contiguous() or batch.dtype != torch.float32:
        raise ValueError("resize_pad_batch expects a contiguous fp32 batch (n,C,H,W)")
    C = batch.shape[1]
    shapes = []
    for im, (oh, ow) in zip(imgs, out_sizes):
        if im.dim() != 3 or im.shape[0] != C:
            raise ValueError("resize_pad_batch: image %s vs %d channels" % (tuple(im.shape), C))
        shapes += [im.shape[1], im.shape[2], int(oh), int(ow)]
    ptrs = (ctypes.c_void_p * n)(*[im.data_ptr() for im in imgs])
    sh = (ctypes.c_int32 * (4 * n))(*shapes)
    with torch.cuda.device(batch.device):
        rc = _lib.load().frcnn_resize_pad_batch_f32(ctypes.cast(ptrs, ctypes.c_void_p), ctypes.cast(sh, ctypes.c_void_p),
                                                    n, C, _ptr(batch), batch.shape[2], batch.shape[3], _stream())
    _lib.check(rc, "resize_pad_batch")
    return batch


def roi_detect_filter(props, regs, scores, row_off, image_sizes, max_rows, score_thresh, min_size):
    """ROIHead/roi_head.py:178-209 for a batch: props (N,4) concatenated, regs (N,K,4) or (N,4K), scores (N,K),
    row_off (B+1) int32, image_sizes (B,2) fp32 (h,w).  -> boxes (B,M,4), scores (B,M), labels (B,M) int32,
    count (B) int32 with M = max_rows*K; the first count[b] rows of image b are its kept candidates in flat order."""
    _need_gpu(props, regs, scores, row_off, image_sizes)
    props, regs, scores = _f32c(props), _f32c(regs), _f32c(scores)
    image_sizes = _f32c(image_sizes)
    row_off = row_off.to(torch.int32).contiguous()
    N, K = scores.shape
    if props.shape != (N, 4) or regs.numel() != N * K * 4 or image_sizes.shape != (row_off.numel() - 1, 2):
        raise ValueError("roi_detect_filter: inconsistent shapes")
    B = row_off.numel() - 1
    M = int(max_rows) * K
    dev = scores.device
    boxes = torch.empty((B, M, 4), dtype=torch.float32, device=dev)
    sc = torch.empty((B, M), dtype=torch.float32, device=dev)
    labels = torch.empty((B, M), dtype=torch.int32, device=dev)
    count = torch.empty((B,), dtype=torch.int32, device=dev)
    with torch.cuda.device(dev):
        rc = _lib.load().frcnn_roi_detect_filter_f32(_ptr(props), _ptr(regs), _ptr(scores), _ptr(row_off),
                                                     _ptr(image_sizes), B, K, int(max_rows), float(score_thresh),
                                                     float(min_size), _ptr(boxes), _ptr(sc), _ptr(labels), _ptr(count),
                                                     _stream())
    _lib.check(rc, "roi_detect_filter")
    return boxes, sc, labels, count


SMOOTH_L1_BETA = 1.0 / 9  # utils.py:315


def rpn_sampled_loss(scores, regs, labels, reg_labels, index, beta=SMOOTH_L1_BETA, want_grad=True):
    """RPN/rpn.py:122-137 in one launch.  scores/labels: (rows) or (B,A); regs/reg_labels: (..,4);
    index: flat int64 rows (b*A + a).  -> (loss (2) [cls, reg], grad_scores, grad_regs)."""
    _need_gpu(scores, regs, labels, reg_labels, index)
    scores, regs, labels, reg_labels = _f32c(scores), _f32c(regs), _f32c(labels), _f32c(reg_labels)
    index = index.to(torch.int64).contiguous()
    rows = scores.numel()
    if regs.numel() != 4 * rows or labels.numel() != rows or reg_labels.numel() != 4 * rows:
        raise ValueError("rpn_sampled_loss: inconsistent shapes")
    loss = torch.empty((2,), dtype=torch.float32, device=scores.device)
    gs = torch.empty_like(scores) if want_grad else None
    gr = torch.empty_like(regs) if want_grad else None
    with torch.cuda.device(scores.device):
        rc = _lib.load().frcnn_rpn_sampled_loss_f32(_ptr(scores), _ptr(regs), _ptr(labels), _ptr(reg_labels),
                                                    _ptr(index), index.numel(), rows, float(beta), _ptr(loss),
                                                    _ptr(gs) if want_grad else None, _ptr(gr) if want_grad else None,
                                                    _stream())
    _lib.check(rc, "rpn_sampled_loss")
    return loss, gs, gr


def roi_loss(logits, pred, cls_label, reg_label, beta=SMOOTH_L1_BETA, want_grad=True):
    """ROIHead/roi_head.py:141-152 in one launch.  logits (N,Kc), pred (N,Kc*4) or (N,Kc,4), cls_label (N) fp32
    class ids, reg_label (N,4).  -> (loss (2) [cls, reg], grad_logits, grad_pred)."""
    _need_gpu(logits, pred, cls_label, reg_label)
    logits, pred, cls_label, reg_label = _f32c(logits), _f32c(pred), _f32c(cls_label), _f32c(reg_label)
    N, Kc = logits.shape
    if pred.numel() != N * Kc * 4 or cls_label.numel() != N or reg_label.numel() != N * 4:
        raise ValueError("roi_loss: inconsistent shapes")
    loss = torch.empty((2,), dtype=torch.float32, device=logits.device)
    gl = torch.empty_like(logits) if want_grad else None
    gp = torch.empty_like(pred) if want_grad else None
    with torch.cuda.device(logits.device):
        rc = _lib.load().frcnn_roi_loss_f32(_ptr(logits), _ptr(pred), _ptr(cls_label), _ptr(reg_label), N, Kc,
                                            float(beta), _ptr(loss), _ptr(gl) if want_grad else None,
                                            _ptr(gp) if want_grad else None, _stream())
    _lib.check(rc, "roi_loss")
    return loss, gl, gp


class RpnSampledLoss(torch.autograd.Function):
    """(cls_loss, reg_loss) of rpn.py:136-137 with gradients to the dense (B,A) scores and (B,A,4) regs."""

    @staticmethod
    def forward(ctx, scores, regs, labels, reg_labels, index):
        need = ctx.needs_input_grad[0] or ctx.needs_input_grad[1]
        loss, gs, gr = rpn_sampled_loss(scores.detach(), regs.detach(), labels, reg_labels, index, want_grad=need)
        if need:
            ctx.save_for_backward(gs, gr)
        return loss[0], loss[1]

    @staticmethod
    def backward(ctx, g_cls, g_reg):
        gs, gr = ctx.saved_tensors
        return (gs * g_cls if ctx.needs_input_grad[0] else None, gr * g_reg if ctx.needs_input_grad[1] else None,
                None, None, None)


class RoiLoss(torch.autograd.Function):
    """(cls_loss, reg_loss) of roi_head.py:144-152 with gradients to the predictor outputs."""

    @staticmethod
    def forward(ctx, logits, pred, cls_label, reg_label):
        need = ctx.needs_input_grad[0] or ctx.needs_input_grad[1]
        loss, gl, gp = roi_loss(logits.detach(), pred.detach(), cls_label, reg_label, want_grad=need)
        if need:
            ctx.save_for_backward(gl, gp)
        return loss[0], loss[1]

    @staticmethod
    def backward(ctx, g_cls, g_reg):
        gl, gp = ctx.saved_tensors
        return (gl * g_cls if ctx.needs_input_grad[0] else None, gp * g_reg if ctx.needs_input_grad[1] else None,
                None, None)


def box_clip(box, image_h, image_w):
    _need_gpu(box)
    box = _f32c(box)
    if box.dim() != 2 or box.shape[1] != 4:
        raise ValueError("box_clip expects (n,4); got %s" % (tuple(box.shape),))
    out = torch.empty_like(box)
    with torch.cuda.device(box.device):
        rc = _lib.load().frcnn_box_clip_f32(_ptr(box), box.shape[0], float(image_h), float(image_w), _ptr(out),
                                            _stream())
    _lib.check(rc, "box_clip")
    return out


def remove_small_box(box, size_thresh):
    """-> (box_out (n,4) [first count rows valid], index (n) int64, count (1) int32 device)."""
    _need_gpu(box)
    box = _f32c(box)
    n = box.shape[0]
    dev = box.device
    box_out = torch.empty_like(box)
    index = torch.empty((n,), dtype=torch.int64, device=dev)
    count = torch.empty((1,), dtype=torch.int32, device=dev)
    with torch.cuda.device(dev):
        rc = _lib.load().frcnn_remove_small_box_f32(_ptr(box), n, float(size_thresh), _ptr(box_out), _ptr(index),
                                                    _ptr(count), _stream())
    _lib.check(rc, "remove_small_box")
    return box_out, index, count


def select_gt(value, thresh):
    """index = where(value > thresh)[0] -> (index (n) int64, count (1) int32 device)."""
    _need_gpu(value)
    value = _f32c(value).reshape(-1)
    n = value.shape[0]
    index = torch.empty((n,), dtype=torch.int64, device=value.device)
    count = torch.empty((1,), dtype=torch.int32, device=value.device)
    with torch.cuda.device(value.device):
        rc = _lib.load().frcnn_select_gt_f32(_ptr(value), n, float(thresh), _ptr(index), _ptr(count), _stream())
    _lib.check(rc, "select_gt")
    return index, count


def decode_clip_filter(anchors, deltas, top_idx, top_score, image_h, image_w, min_size):
    """Fused RPN/rpn.py:67-83 for a batch.  anchors (A,4) shared or (B,A,4); deltas (B,A,4);
    top_idx / top_score (B,k).  -> boxes (B,k,4), scores (B,k), src (B,k) int32, count (B) int32."""
    _need_gpu(anchors, deltas, top_idx, top_score)
    anchors, deltas, top_score = _f32c(anchors), _f32c(deltas), _f32c(top_score)
    top_idx = top_idx.contiguous()
    if top_idx.dtype != torch.int32:
        top_idx = top_idx.to(torch.int32)
    B, A = deltas.shape[0], deltas.shape[1]
    k = top_idx.shape[1]
    if anchors.dim() == 2:
        stride = 0
        if anchors.shape[0] != A:
            raise ValueError("anchors (%d) and deltas (%d) disagree" % (anchors.shape[0], A))
    else:
        stride = A * 4
        if anchors.shape[0] != B or anchors.shape[1] != A:
            raise ValueError("anchors %s vs deltas %s" % (tuple(anchors.shape), tuple(deltas.shape)))
    dev = deltas.device
    boxes = torch.empty((B, k, 4), dtype=torch.float32, device=dev)
    scores = torch.empty((B, k), dtype=torch.float32, device=dev)
    src = torch.empty((B, k), dtype=torch.int32, device=dev)
    count = torch.empty((B,), dtype=torch.int32, device=dev)
    with torch.cuda.device(dev):
        rc = _lib.load().frcnn_decode_clip_filter_f32(
            _ptr(anchors), stride, _ptr(deltas), _ptr(top_idx), _ptr(top_score), B, A, k, float(image_h),
            float(image_w), float(min_size), _ptr(boxes), _ptr(scores), _ptr(src), _ptr(count), _stream())
    _lib.check(rc, "decode_clip_filter")
    return boxes, scores, src, count


# --------------------------------------------------------------------------------------- K4 NMS
# Pinned host words that kernels write directly (NmsRounds): never handed back to torch's pinned-memory cache, because a
# launch that is still queued when its owner is dropped would then write into whatever tensor gets the block next.
_PINNED_FOREVER = []


class NmsRounds:
    """How far into the round-path NMS the caller's recent batches got, fed forward as the next call's launch bound
    (frcnn_nms_sorted_rounds_f32).  The kernels leave, per image, the count of 64-candidate blocks that had work (16
    per round) in pinned host memory that the GPU writes directly; the host reads whatever has landed -- the counts
    of the last call that FINISHED, never a synchronisation -- and asks for their maximum plus `slack` blocks (4 = a
    quarter of a round: a batch that gets that much further still finishes inside the bound; one that gets further
    yet is finished by the last round's tail, correct and slower).  Until a first call has finished
    every round is enqueued, as without it.  Keep lists do not depend on the bound; one object per call site and
    stream."""

    UNKNOWN = 1 << 20

    def __init__(self, slack=4, history=8):
        self.slack = int(slack)
        self.history = int(history)
        self._used = {}
        self._seen = {}

    def _slot(self, key, B):
        t = self._used.get(key)
        if t is None:
            t = torch.full((B,), self.UNKNOWN, dtype=torch.int32).pin_memory()
            _PINNED_FOREVER.append(t)  # a few bytes per call site; see the note at _PINNED_FOREVER
            self._used[key] = t
            self._seen[key] = collections.deque(maxlen=self.history)
        return t

    def bound(self, key, B):
        """-> (max_blocks argument, pinned tensor the call reports into).  The bound covers the furthest any of the
        last `history` observations got, plus the slack: batches whose reach wanders stay inside it."""
        t = self._slot(key, B)
        m = int(t.max())
        if m >= self.UNKNOWN:
            return 0, t
        seen = self._seen[key]
        seen.append(m)
        return max(1, max(seen) + self.slack), t


def nms_sorted(boxes, n_per_image, iou_threshold, max_keep, rounds=None):
    """Batched greedy NMS over rows already in descending-score order.
    boxes (B,n,4); n_per_image (B) int32 device or None.  -> keep (B,max_keep) int32, n_keep (B).
    rounds: an NmsRounds that bounds the launches by what earlier batches needed (same result), or None."""
    _need_gpu(boxes, n_per_image)
    boxes = _f32c(boxes)
    B, n = boxes.shape[0], boxes.shape[1]
    dev = boxes.device
    max_keep = int(max_keep)
    keep = torch.empty((B, max(max_keep, 1)), dtype=torch.int32, device=dev)
    n_keep = torch.empty((B,), dtype=torch.int32, device=dev)
    lib = _lib.load()
    nbytes = lib.frcnn_nms_workspace_bytes(B, n)  # 0 for small n (single-launch path)
    ws = torch.empty((max(nbytes, 16),), dtype=torch.uint8, device=dev)
    if n_per_image is not None and n_per_image.dtype != torch.int32:
        n_per_image = n_per_image.to(torch.int32)
    with torch.cuda.device(dev):
        if rounds is not None and nbytes > 0 and B > 0:
            max_blocks, used = rounds.bound((dev.index, B, n, max_keep, float(iou_threshold)), B)
            rc = lib.frcnn_nms_sorted_rounds_f32(_ptr(boxes), _ptr(n_per_image), B, n, float(iou_threshold), max_keep,
                                                 _ptr(keep), _ptr(n_keep), _ptr(ws), nbytes, max_blocks,
                                                 used.data_ptr(), _stream())
        else:
            rc = lib.frcnn_nms_sorted_f32(_ptr(boxes), _ptr(n_per_image), B, n, float(iou_threshold), max_keep,
                                          _ptr(keep), _ptr(n_keep), _ptr(ws), nbytes, _stream())
    _lib.check(rc, "nms_sorted")
    return keep[:, :max_keep], n_keep


def gather_boxes(src, idx, count=None):
    """out[b,j] = src[b, idx[b,j]] for j < count[b], zero rows after.  src (B,n,4); idx (B,m) int32."""
    _need_gpu(src, idx, count)
    src = _f32c(src)
    idx = idx.contiguous()
    B, n = src.shape[0], src.shape[1]
    m = idx.shape[1]
    out = torch.empty((B, m, 4), dtype=torch.float32, device=src.device)
    with torch.cuda.device(src.device):
        rc = _lib.load().frcnn_gather_boxes_f32(_ptr(src), _ptr(idx), _ptr(count), B, n, m, _ptr(out), _stream())
    _lib.check(rc, "gather_boxes")
    return out


def nms(boxes, scores, iou_threshold):
    """torchvision.ops.nms(boxes, scores, iou_threshold) -> int64 indices of kept boxes in
    descending-score order (call sites RPN/rpn.py:84, ROIHead/roi_head.py:215)."""
    _need_gpu(boxes, scores)
    n = boxes.shape[0]
    if n == 0:
        return torch.empty((0,), dtype=torch.int64, device=boxes.device)
    if boxes.dim() != 2 or boxes.shape[1] != 4 or scores.dim() != 1 or scores.shape[0] != n:
        raise ValueError("nms expects boxes (n,4) and scores (n,); got %s, %s" % (tuple(boxes.shape), tuple(scores.shape)))
    _, order = topk_desc(scores.reshape(1, n), n, want_values=False)
    sorted_boxes = gather_boxes(boxes.reshape(1, n, 4), order)
    keep, n_keep = nms_sorted(sorted_boxes, None, iou_threshold, n)
    cnt = int(n_keep.item())
    return order[0, keep[0, :cnt].long()].long()


# ----------------------------------------------------------------------- K5 IoU, target labels
def box_iou(box1, box2):
    _need_gpu(box1, box2)
    box1, box2 = _f32c(box1), _f32c(box2)
    n, m = box1.shape[0], box2.shape[0]
    out = torch.empty((n, m), dtype=torch.float32, device=box1.device)
    with torch.cuda.device(box1.device):
        rc = _lib.load().frcnn_box_iou_f32(_ptr(box1), n, _ptr(box2), m, _ptr(out), _stream())
    _lib.check(rc, "box_iou")
    return out


def iou_label_encode(box1, box2, m_per_image, neg_threshold, pos_threshold, labels=None, weights=None,
                     want=("label", "argmax", "max_iou", "dev")):
    """Fused tagging_box + box_deviation for a batch.
    box1 (N,4) shared or (B,N,4); box2 (B,Mmax,4); m_per_image (B) int32 device or None;
    labels (B,Mmax) fp32 or None; weights: 4 host floats or None.
    -> dict with the requested outputs: label (B,N), argmax (B,N) int32, max_iou (B,N), dev (B,N,4)."""
    _need_gpu(box1, box2, m_per_image, labels)
    box1, box2 = _f32c(box1), _f32c(box2)
    B, m_max = box2.shape[0], box2.shape[1]
    if m_max == 0:
        raise ValueError("box_2 is empty: the reference's iou.max(dim=1) raises on an (N,0) matrix")
    if box1.dim() == 2:
        N, stride = box1.shape[0], 0
    else:
        N, stride = box1.shape[1], box1.shape[1] * 4
        if box1.shape[0] != B:
            raise ValueError("box1 batch %d vs box2 batch %d" % (box1.shape[0], B))
    dev = box2.device
    if labels is not None:
        labels = _f32c(labels)
    if m_per_image is not None and m_per_image.dtype != torch.int32:
        m_per_image = m_per_image.to(torch.int32)
    out = {}
    if "label" in want:
        out["label"] = torch.empty((B, N), dtype=torch.float32, device=dev)
    if "argmax" in want:
        out["argmax"] = torch.empty((B, N), dtype=torch.int32, device=dev)
    if "max_iou" in want:
        out["max_iou"] = torch.empty((B, N), dtype=torch.float32, device=dev)
    if "dev" in want:
        out["dev"] = torch.empty((B, N, 4), dtype=torch.float32, device=dev)
    if weights is not None:
        wa, wp = _host_f32([float(w) for w in weights])
    else:
        wa, wp = None, ctypes.c_void_p(0)
    with torch.cuda.device(dev):
        rc = _lib.load().frcnn_iou_label_encode_f32(
            _ptr(box1), stride, _ptr(box2), _ptr(m_per_image), _ptr(labels), B, N, m_max,
            float(np.float32(neg_threshold)), float(np.float32(pos_threshold)), wp, _ptr(out.get("label")),
            _ptr(out.get("argmax")), _ptr(out.get("max_iou")), _ptr(out.get("dev")), _stream())
    _lib.check(rc, "iou_label_encode")
    return out


# ----------------------------------------------------------------------------- K6/K7 RoI ops
def sample_rows(pos_mask, neg_mask, num_sample, pos_fraction):
    """The random sampling of RPN/rpn.py:115-122 and ROIHead/roi_head.py:113-121 for a whole batch.

    pos_mask / neg_mask: (B, N) bool on the device -- the rows `torch.where(label == 1)` / `(label == 0)` list
    per image.  Returns (flat (S,) int64 = b * N + row, sizes: list of B ints): per image its sampled NEGATIVES
    first, then its positives (rpn.py:122), images in order.  What must stay per image stays per image:
    utils.get_sampling_factor draws `torch.randperm(pos_num)` then `torch.randperm(neg_num)` on the CPU's global
    generator in the reference's order (RNG parity under torch.manual_seed).  Everything else is batched: ONE
    host read (the B x 2 counts), ONE host-to-device copy (ranks + order), and the k-th listed row of an image is
    found by a search in the running count of its mask -- no nonzero(), no per-image gathers."""
    from .utils import get_sampling_factor
    B, N = pos_mask.shape
    dev = pos_mask.device
    cum_pos = pos_mask.cumsum(1, dtype=torch.int32)
    cum_neg = neg_mask.cumsum(1, dtype=torch.int32)
    counts = torch.stack([cum_pos[:, -1], cum_neg[:, -1]], 1).tolist() if N else [[0, 0]] * B   # the one host read
    factors = [get_sampling_factor(num_sample, pos_fraction, n_pos, n_neg) for n_pos, n_neg in counts]
    s_pos = max([f[0].numel() for f in factors] + [1])
    s_neg = max([f[1].numel() for f in factors] + [1])
    sizes = [f[0].numel() + f[1].numel() for f in factors]
    # one host buffer: (B, s_neg) ranks of the negatives, (B, s_pos) ranks of the positives (1-based: the value
    # the running count reaches AT the wanted row), then for every sampled row its place in those two matrices
    host = torch.ones(B * (s_neg + s_pos) + sum(sizes), dtype=torch.int32)
    ranks = host[:B * (s_neg + s_pos)].view(B, s_neg + s_pos)
    order = host[B * (s_neg + s_pos):]
    at = 0
    for b, (pos_f, neg_f) in enumerate(factors):
        n_n, n_p = neg_f.numel(), pos_f.numel()
        ranks[b, :n_n] = neg_f + 1
        ranks[b, s_neg:s_neg + n_p] = pos_f + 1
        order[at:at + n_n] = torch.arange(b * (s_neg + s_pos), b * (s_neg + s_pos) + n_n)
        order[at + n_n:at + n_n + n_p] = torch.arange(b * (s_neg + s_pos) + s_neg, b * (s_neg + s_pos) + s_neg + n_p)
        at += n_n + n_p
    host = host.to(dev, non_blocking=True)
    ranks = host[:B * (s_neg + s_pos)].view(B, s_neg + s_pos)
    order = host[B * (s_neg + s_pos):].long()
    rows = torch.cat([torch.searchsorted(cum_neg, ranks[:, :s_neg].contiguous()),
                      torch.searchsorted(cum_pos, ranks[:, s_neg:].contiguous())], 1)
    rows = rows.clamp_(max=max(N - 1, 0)) + torch.arange(B, device=dev)[:, None] * N
    return rows.reshape(-1)[order], sizes


def build_rois(props, count=None):
    """(B,P,4) padded proposals + per-image counts -> rois (B*P,5) compacted, total (1) int32 device."""
    _need_gpu(props, count)
    props = _f32c(props)
    B, P = props.shape[0], props.shape[1]
    rois = torch.empty((B * P, 5), dtype=torch.float32, device=props.device)
    total = torch.empty((1,), dtype=torch.int32, device=props.device)
    with torch.cuda.device(props.device):
        rc = _lib.load().frcnn_build_rois_f32(_ptr(props), _ptr(count), B, P, _ptr(rois), _ptr(total), _stream())
    _lib.check(rc, "build_rois")
    return rois, total


def level_map(rois, k_min, k_max, n_rois=None):
    _need_gpu(rois, n_rois)
    rois = _f32c(rois)
    K = rois.shape[0]
    lvl = torch.full((K,), -1, dtype=torch.int32, device=rois.device)
    with torch.cuda.device(rois.device):
        rc = _lib.load().frcnn_level_map_f32(_ptr(rois), _ptr(n_rois), K, int(k_min), int(k_max), _ptr(lvl), _stream())
    _lib.check(rc, "level_map")
    return lvl


def roi_align(feat, rois, output_size, spatial_scale, sampling_ratio, n_rois=None, lvl=None, lvl_value=0, out=None):
    """torchvision roi_align(aligned=False) on one level.  feat (B,C,H,W); rois (K,5) -> (K,C,ph,pw).
    With `out` given, only rows selected by lvl == lvl_value (and < n_rois) are written."""
    _need_gpu(feat, rois, n_rois, lvl, out)
    feat, rois = _f32c(feat), _f32c(rois)
    B, C, H, W = feat.shape
    K = rois.shape[0]
    ph, pw = int(output_size[0]), int(output_size[1])
    if out is None:
        # rows past *n_rois are never written; only a level-filtered call needs a zero background
        alloc = torch.zeros if lvl is not None else torch.empty
        out = alloc((K, C, ph, pw), dtype=torch.float32, device=feat.device)
    with torch.cuda.device(feat.device):
        rc = _lib.load().frcnn_roi_align_f32(_ptr(feat), B, C, H, W, _ptr(rois), _ptr(n_rois), K, ph, pw,
                                             float(spatial_scale), int(sampling_ratio), _ptr(lvl), int(lvl_value),
                                             _ptr(out), _stream())
    _lib.check(rc, "roi_align")
    return out


def roi_pool(feat, rois, output_size, spatial_scale):
    """torchvision roi_pool (max) -> (out (K,C,ph,pw), argmax (K,C,ph,pw) int32)."""
    _need_gpu(feat, rois)
    feat, rois = _f32c(feat), _f32c(rois)
    B, C, H, W = feat.shape
    K = rois.shape[0]
    ph, pw = int(output_size[0]), int(output_size[1])
    out = torch.empty((K, C, ph, pw), dtype=torch.float32, device=feat.device)
    arg = torch.empty((K, C, ph, pw), dtype=torch.int32, device=feat.device)
    with torch.cuda.device(feat.device):
        rc = _lib.load().frcnn_roi_pool_f32(_ptr(feat), B, C, H, W, _ptr(rois), K, ph, pw, float(spatial_scale),
                                            _ptr(out), _ptr(arg), _stream())
    _lib.check(rc, "roi_pool")
    return out, arg


def roi_pool_batched(feat, props, count, output_size, spatial_scale):
    """torchvision roi_pool (max) over zero-padded proposals (B,P,4) with per-image counts (B) int32 or None.
    -> (out (B*P,C,7,7), argmax (B*P,C,7,7) int32, total (1) int32); the first sum(count) rows are valid, in image
    order.  Planes stay resident in LDS (7 x 7 bins, maps up to about 37 x 64 at 16 channels a time)."""
    _need_gpu(feat, props, count)
    feat, props = _f32c(feat), _f32c(props)
    B, C, H, W = feat.shape
    if props.dim() != 3 or props.shape[0] != B or props.shape[2] != 4:
        raise ValueError("roi_pool_batched expects props (B,P,4); got %s for B = %d" % (tuple(props.shape), B))
    P = props.shape[1]
    if count is not None and count.dtype != torch.int32:
        count = count.to(torch.int32)
    ph, pw = int(output_size[0]), int(output_size[1])
    out = torch.empty((B * P, C, ph, pw), dtype=torch.float32, device=feat.device)
    arg = torch.empty((B * P, C, ph, pw), dtype=torch.int32, device=feat.device)
    total = torch.empty((1,), dtype=torch.int32, device=feat.device)
    with torch.cuda.device(feat.device):
        rc = _lib.load().frcnn_roi_pool_batched_f32(_ptr(feat), B, C, H, W, _ptr(props), _ptr(count), P, ph, pw,
                                                    float(spatial_scale), _ptr(out), _ptr(arg), _ptr(total), _stream())
    _lib.check(rc, "roi_pool_batched")
    return out, arg, total


def infer_scale(feature_hw, image_hw):
    """torchvision poolers._infer_scale: 2 ** round(log2(fp32(feat/img))); both axes must agree."""
    scales = []
    for s1, s2 in zip(feature_hw, image_hw):
        approx = np.float32(float(s1) / float(s2))
        scales.append(2.0 ** float(np.round(np.log2(approx))))
    if scales[0] != scales[1]:
        raise AssertionError("feature map and image disagree on the scale per axis: %r" % (scales,))
    return scales[0]


# Which kernels pool a pyramid: "cl" = lanes-are-channels on channel-innermost maps (csrc/roi_cl.hip), "tiles" = LDS
# tiles of NCHW maps (csrc/roi_tile.hip).  "auto" takes cl for maps that already are channels-last (read in place:
# 0.84 ms against 0.82 + a 0.15 ms copy at BASELINE configs[4]) and tiles for NCHW maps (cl would first copy them:
# 0.99 ms); DESIGN.md section 4 has the measurements.
ROI_LEVELS_PATH = os.environ.get("FRCNN_ROI_LEVELS_PATH", "auto")
_cl_workspaces = {}


def _cl_workspace(dev, nbytes):
    """One workspace per (device, stream): calls on a stream are ordered, so the next call may overwrite it."""
    key = (dev.index, torch.cuda.current_stream(dev).cuda_stream)
    ws = _cl_workspaces.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = torch.empty((max(int(nbytes), 256),), dtype=torch.uint8, device=dev)
        _cl_workspaces[key] = ws
    return ws


def _is_channels_last(f):
    return f.dim() == 4 and f.is_contiguous(memory_format=torch.channels_last) and not f.is_contiguous()


def _roi_align_levels(cfg, props, count, feats, path=None):
    """Forward of every level: (out (B*P, C, oh, ow), total (1) int32)."""
    output_size, sampling_ratio, scales, k_min, k_max = cfg
    B, P = props.shape[0], props.shape[1]
    C = feats[0].shape[1]
    dev = props.device
    out = torch.empty((B * P, C) + tuple(output_size), dtype=torch.float32, device=dev)
    total = torch.empty((1,), dtype=torch.int32, device=dev)
    for l, f in enumerate(feats):
        if f.shape[0] != B or f.shape[1] != C:
            raise ValueError("feature map %d has shape %s, expected (%d,%d,h,w)" % (l, tuple(f.shape), B, C))
    n = len(feats)
    hw = (ctypes.c_int32 * (2 * n))(*[int(v) for f in feats for v in f.shape[2:]])
    sc = (ctypes.c_float * n)(*[float(s) for s in scales])
    lib = _lib.load()
    path = path or ROI_LEVELS_PATH
    cl_maps = all(f.dtype == torch.float32 and _is_channels_last(f) for f in feats)
    if path == "auto":
        fits_plane = n == 1 and feats[0].shape[2] * ((feats[0].shape[3] + 15) // 16 * 16) * 64 <= 150 * 1024
        path = "cl" if cl_maps and not fits_plane else "tiles"
    if path == "cl" and tuple(output_size) == (7, 7) and sampling_ratio == 2 and P > 0:
        nbytes = lib.frcnn_roi_align_levels_cl_workspace_bytes(hw, n, B, C, P, int(cl_maps))
        if nbytes > 0:
            feats = [f if cl_maps else _f32c(f) for f in feats]
            ws = _cl_workspace(dev, nbytes)
            ptrs = (ctypes.c_void_p * n)(*[f.data_ptr() for f in feats])
            with torch.cuda.device(dev):
                rc = lib.frcnn_roi_align_levels_cl_f32(
                    ptrs, hw, sc, n, B, C, int(cl_maps), _ptr(props), _ptr(count), P, 7, 7, 2, k_min, k_max,
                    _ptr(out), _ptr(total), _ptr(ws), ws.numel(), _stream())
                _lib.check(rc, "roi_align_levels_cl")
            return out, total
    feats = [_f32c(f) for f in feats]
    ptrs = (ctypes.c_void_p * n)(*[f.data_ptr() for f in feats])
    with torch.cuda.device(dev):
        rc = lib.frcnn_roi_align_levels_f32(
            ptrs, hw, sc, n, B, C, _ptr(props), _ptr(count), P, output_size[0], output_size[1], sampling_ratio,
            k_min, k_max, _ptr(out), _ptr(total), _stream())
        _lib.check(rc, "roi_align_levels")
    return out, total


def roi_align_levels_backward(cfg, props, count, grad_out, feat_shapes, wanted=None):
    """Gradients of _roi_align_levels with respect to each feature map (None where not wanted)."""
    output_size, sampling_ratio, scales, k_min, k_max = cfg
    B, P = props.shape[0], props.shape[1]
    grad_out = _f32c(grad_out)
    grads = []
    lib = _lib.load()
    with torch.cuda.device(props.device):
        for l, (shape, s) in enumerate(zip(feat_shapes, scales)):
            if wanted is not None and not wanted[l]:
                grads.append(None)
                continue
            g = torch.empty(tuple(shape), dtype=torch.float32, device=props.device)
            rc = lib.frcnn_roi_align_batched_backward_f32(
                _ptr(grad_out), B, shape[1], shape[2], shape[3], _ptr(props), _ptr(count), P, output_size[0],
                output_size[1], float(s), sampling_ratio, l, len(feat_shapes), k_min, k_max, _ptr(g), _stream())
            _lib.check(rc, "roi_align_batched_backward")
            grads.append(g)
    return grads


class _RoIAlignLevels(torch.autograd.Function):
    """MultiScaleRoIAlign over padded proposals, differentiable in the feature maps: forward and backward are
    the HIP kernels (ROIHead/roi_head.py:127-130 under autograd).  Boxes get no gradient, as in torchvision."""

    @staticmethod
    def forward(ctx, cfg, props, count, *feats):
        ctx.cfg = cfg
        ctx.feat_shapes = [tuple(f.shape) for f in feats]
        ctx.save_for_backward(props, count) if count is not None else ctx.save_for_backward(props)
        ctx.has_count = count is not None
        out, total = _roi_align_levels(cfg, props, count, feats)
        ctx.mark_non_differentiable(total)
        return out, total

    @staticmethod
    def backward(ctx, grad_out, _grad_total):
        saved = ctx.saved_tensors
        props, count = (saved[0], saved[1]) if ctx.has_count else (saved[0], None)
        grads = roi_align_levels_backward(ctx.cfg, props, count, grad_out, ctx.feat_shapes, ctx.needs_input_grad[3:])
        return (None, None, None) + tuple(grads)


class MultiScaleRoIAlign(torch.nn.Module):
    """torchvision.ops.MultiScaleRoIAlign(featmap_names, output_size, sampling_ratio) as the
    reference uses it (ROIHead/roi_pooling.py:44-53): FPN level mapper + RoIAlign per level.

    forward(x: dict[str, Tensor(B,C,h,w)], boxes: list[Tensor(P_i,4)], image_shapes: list[(h,w)])
    -> Tensor(sum P_i, C, oh, ow).  `forward_padded` is the sync-free batched form."""

    def __init__(self, featmap_names, output_size, sampling_ratio, *, canonical_scale=224, canonical_level=4):
        super().__init__()
        if isinstance(output_size, int):
            output_size = (output_size, output_size)
        self.featmap_names = list(featmap_names)
        self.output_size = tuple(output_size)
        self.sampling_ratio = sampling_ratio
        if canonical_scale != 224 or canonical_level != 4:
            raise ValueError("only the canonical (224, 4) level mapper is built into the kernel")

    def _levels(self, x, image_shapes):
        feats = [v for k, v in x.items() if k in self.featmap_names]
        if not feats:
            raise ValueError("none of the feature maps %r is in featmap_names %r" % (list(x), self.featmap_names))
        max_h = max(s[0] for s in image_shapes)
        max_w = max(s[1] for s in image_shapes)
        scales = [infer_scale(f.shape[-2:], (max_h, max_w)) for f in feats]
        k_min = int(-math.log2(scales[0]))
        k_max = int(-math.log2(scales[-1]))
        return feats, scales, k_min, k_max

    def _pool_padded(self, feats, scales, k_min, k_max, props, count):
        """One batched launch per level over zero-padded proposals; rows compacted in image order.
        Differentiable with respect to the feature maps (as torchvision's op is) when any of them requires grad."""
        cfg = (self.output_size, int(self.sampling_ratio), tuple(float(s) for s in scales), int(k_min), int(k_max))
        if torch.is_grad_enabled() and any(f.requires_grad for f in feats):
            return _RoIAlignLevels.apply(cfg, props, count, *feats)
        return _roi_align_levels(cfg, props, count, feats)

    def forward(self, x, boxes, image_shapes):
        feats, scales, k_min, k_max = self._levels(x, image_shapes)
        dev = feats[0].device
        _need_gpu(*feats)
        B = feats[0].shape[0]
        C = feats[0].shape[1]
        if len(boxes) > B:
            raise ValueError("%d box lists for a batch of %d feature maps" % (len(boxes), B))
        counts = [int(b.shape[0]) for b in boxes] + [0] * (B - len(boxes))
        total = sum(counts)
        if total == 0:
            return torch.zeros((0, C) + self.output_size, device=dev)
        P = max(counts)
        props = torch.zeros((B, P, 4), dtype=torch.float32, device=dev)
        for i, b in enumerate(boxes):
            if counts[i]:
                props[i, :counts[i]] = b.detach().to(device=dev, dtype=torch.float32).reshape(-1, 4)
        count = torch.tensor(counts, dtype=torch.int32, device=dev)
        out, _ = self._pool_padded(feats, scales, k_min, k_max, props, count)
        return out[:total]

    def forward_padded(self, x, props, count, image_shapes):
        """props (B,P,4) zero-padded, count (B) int32 device (or None = P each) -> (B*P, C, oh, ow)
        whose first sum(count) rows are valid (same row order as forward), plus the device-side
        total.  No host sync, no intermediate roi list."""
        feats, scales, k_min, k_max = self._levels(x, image_shapes)
        _need_gpu(props, count, *feats)
        if count is not None and count.dtype != torch.int32:
            count = count.to(torch.int32)
        return self._pool_padded(feats, scales, k_min, k_max, _f32c(props), count)


# ------------------------------------------------------- 8-bit dense layers of the box head
_I8_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
I8_MAX_K = 131071  # the 32-bit sums of the product cannot wrap up to here
I8_MAX_ROW = 1 << 30  # longest row of the quantiser alone
I8_MAX_ROWS = 4194303  # rows of any matrix

# A layer of a few rows is bound by the host, so these wrappers spend little there: pointers go to ctypes as numbers, the
# stream comes as a number without a Stream object around it (0.1 us against 1.9), the device is switched only if it is
# another one, and tensors that already have the right form are not touched.


def _i8_call(name, dev, *args):
    """One entry point on dev's current stream."""
    index, fn = dev.index, getattr(_lib.load(), name)
    if torch.cuda.current_device() == index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc != 0:
        _lib.check(rc, name)


@functools.lru_cache(maxsize=1024)
def _i8_bytes(name, M, N, K):
    return getattr(_lib.load(), name)(M, N, K)


def _i8_workspace(name, M, N, K, dev):
    """-> (tensor or None, address or None, bytes): a fresh one for every call (the caching allocator ties it to the current
    stream or graph), none where the call needs none."""
    nbytes = _i8_bytes(name, M, N, K)
    if nbytes == 0:
        return None, None, 0
    ws = torch.empty((nbytes,), dtype=torch.uint8, device=dev)
    return ws, ws.data_ptr(), nbytes


def _at(t):
    return t.data_ptr() if t is not None else None


def _i8_device(what, dev, *tensors):
    for t in tensors:
        if t is not None and t.device != dev:
            _need_gpu(t)
            raise ValueError("%s: all tensors have to be on %s; got one on %s" % (what, dev, t.device))


def _i8_sizes(what, M, N, K, longest=I8_MAX_K):
    """Before a copy, an allocation or a call: ctypes would pass on the low 32 bits of a larger number."""
    if M > I8_MAX_ROWS or N > I8_MAX_ROWS or K > longest:
        raise ValueError("%s: %d rows by %d channels, rows of %d; at most %d, %d and %d"
                         % (what, M, N, K, I8_MAX_ROWS, I8_MAX_ROWS, longest))


def _i8_rows(x, what, longest=I8_MAX_K):
    """x (M,K) as a tensor the kernels read in place: one of the three float types, elements of a row next to each
    other, rows any stride apart."""
    if not x.is_cuda:
        _need_gpu(x)
    if x.dim() != 2 or x.shape[1] == 0:
        raise ValueError("%s expects (M,K) with K > 0; got %s" % (what, tuple(x.shape)))
    _i8_sizes(what, x.shape[0], 1, x.shape[1], longest)
    if x.dtype not in _I8_TYPES:
        x = x.detach().to(torch.float32)
    return x if x.stride(1) == 1 or x.shape[1] == 1 else x.detach().contiguous()


def _row_stride(t):
    """Row stride of a 2-d tensor whose rows are contiguous.  (torch leaves the stride of a single row arbitrary.)"""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _i8_codes(codes):
    return codes if codes.stride(1) == 1 or codes.shape[1] == 1 else codes.contiguous()


def _f32v(t):
    """A vector as the kernels read it."""
    return t if t is None or (t.dtype == torch.float32 and t.is_contiguous()) else t.detach().to(torch.float32).contiguous()


def _i8_count(n_rows, what, dev):
    if n_rows is None:
        return None
    _i8_device(what, dev, n_rows)
    if n_rows.numel() != 1:
        raise ValueError("%s: n_rows expects one element; got %s" % (what, tuple(n_rows.shape)))
    if n_rows.dtype in (torch.int64, torch.float32, torch.float64):
        n_rows = n_rows.clamp(0, I8_MAX_ROWS)  # to within 32 bits, not to their low half
    return n_rows if n_rows.dtype == torch.int32 else n_rows.to(torch.int32)


def _i8_weights(codes, scale, bias, K, dev, what):
    _i8_device(what, dev, codes, scale, bias)
    if codes.dtype != torch.int8 or codes.dim() != 2 or codes.shape[0] == 0 or codes.shape[1] != K:
        raise ValueError("%s expects weight codes (N,%d) int8; got %s %s" % (what, K, tuple(codes.shape), codes.dtype))
    N = codes.shape[0]
    _i8_sizes(what, 0, N, K)
    if scale.dim() != 1 or scale.shape[0] != N or (bias is not None and (bias.dim() != 1 or bias.shape[0] != N)):
        raise ValueError("%s expects a scale and a bias for each of the %d outputs" % (what, N))
    return N, _i8_codes(codes), _f32v(scale), _f32v(bias)


def quantize_rows_i8(x, n_rows=None):
    """Rows of x (M,K; fp32, bf16 or fp16) as 8-bit integers: scale (M) = max |x| / 127 in fp32, codes (M,K) int8 = the
    whole numbers nearest to 127 x / max |x| (of the exact quotient, ties to even), so that x ~ codes * scale[:, None].
    At most 4,194,303 rows of up to 2^30 elements.
    A row of zeros: scale 0, codes 0; a row with an Inf or a NaN: scale NaN, codes 0.  n_rows (1) int32 on the device:
    rows behind it are left out (their outputs are unspecified), as in the padded RoI path.  Rows of the codes lie a
    multiple of 16 bytes apart, the form matmul_i8 reads in place."""
    x = _i8_rows(x, "quantize_rows_i8", I8_MAX_ROW)
    M, K = x.shape
    dev = x.device
    n_rows = _i8_count(n_rows, "quantize_rows_i8", dev)
    kp = (K + 15) // 16 * 16
    codes = torch.empty((M, kp), dtype=torch.int8, device=dev)
    scale = torch.empty((M,), dtype=torch.float32, device=dev)
    _i8_call("frcnn_quantize_rows_i8", dev, x.data_ptr(), _I8_TYPES[x.dtype], _row_stride(x), M, K, _at(n_rows),
             codes.data_ptr(), kp, scale.data_ptr())
    return (codes if kp == K else codes[:, :K]), scale


def matmul_i8(codes, scale, weight_codes, weight_scale, bias=None, relu=False, out_dtype=torch.float32, n_rows=None):
    """out (M,N) = (codes @ weight_codes^T) * scale[:, None] * weight_scale + bias, then max(., 0) if relu: the product
    of two row-quantised matrices (quantize_rows_i8), its sums exact, the rest in 64 bits, rounded to out_dtype.  With relu
    a positive result that out_dtype rounds to zero is -0.0, which is how linear_i8_backward knows it."""
    _need_gpu(codes, scale)
    if codes.dtype != torch.int8 or codes.dim() != 2 or codes.shape[1] == 0 or scale.shape != (codes.shape[0],):
        raise ValueError("matmul_i8 expects codes (M,K) int8 and a scale for each row; got %s %s, %s"
                         % (tuple(codes.shape), codes.dtype, tuple(scale.shape)))
    if out_dtype not in _I8_TYPES:
        raise ValueError("matmul_i8: out_dtype is float32, bfloat16 or float16; got %s" % out_dtype)
    M, K = codes.shape
    _i8_sizes("matmul_i8", M, 1, K)
    dev = codes.device
    _i8_device("matmul_i8", dev, scale)
    N, weight_codes, weight_scale, bias = _i8_weights(weight_codes, weight_scale, bias, K, dev, "matmul_i8")
    codes, scale, n_rows = _i8_codes(codes), _f32v(scale), _i8_count(n_rows, "matmul_i8", dev)
    out = torch.empty((M, N), dtype=out_dtype, device=dev)
    ws, ws_at, nbytes = _i8_workspace("frcnn_matmul_i8_workspace_bytes", M, N, K, dev)
    _i8_call("frcnn_matmul_i8", dev, codes.data_ptr(), _row_stride(codes), scale.data_ptr(), weight_codes.data_ptr(),
             _row_stride(weight_codes), weight_scale.data_ptr(), _at(bias), 1 if relu else 0, M, N, K, _at(n_rows),
             out.data_ptr(), _I8_TYPES[out_dtype], N, ws_at, nbytes)
    return out


def linear_i8(x, weight_codes, weight_scale, bias=None, relu=False, out_dtype=None, n_rows=None):
    """A served dense layer: quantize_rows_i8(x) and matmul_i8 in one call.  x (M,K) fp32, bf16 or fp16; weight_codes
    (N,K) int8 and weight_scale (N) from quantize_rows_i8(weight); -> (M,N) in out_dtype (x's type by default).
    n_rows (1) int32 on the device: rows behind it are neither read nor written.  The result is detached; FrozenLinearI8
    also has the gradient of x, LinearI8 trains the weights."""
    x = _i8_rows(x, "linear_i8")
    M, K = x.shape
    dev = x.device
    if out_dtype is None:
        out_dtype = x.dtype
    elif out_dtype not in _I8_TYPES:
        raise ValueError("linear_i8: out_dtype is float32, bfloat16 or float16; got %s" % out_dtype)
    N, weight_codes, weight_scale, bias = _i8_weights(weight_codes, weight_scale, bias, K, dev, "linear_i8")
    n_rows = _i8_count(n_rows, "linear_i8", dev)
    out = x.new_empty((M, N), dtype=out_dtype)
    ws, ws_at, nbytes = _i8_workspace("frcnn_linear_i8_workspace_bytes", M, N, K, dev)
    _i8_call("frcnn_linear_i8", dev, x.data_ptr(), _I8_TYPES[x.dtype], _row_stride(x), weight_codes.data_ptr(),
             _row_stride(weight_codes), weight_scale.data_ptr(), _at(bias), 1 if relu else 0, M, N, K, _at(n_rows),
             out.data_ptr(), _I8_TYPES[out_dtype], N, ws_at, nbytes)
    return out


def linear_i8_backward(grad, y, codes, scale, weight_codes, weight_scale, x_dtype=torch.float32,
                       weight_dtype=torch.float32, want=(True, True, True)):
    """Straight-through gradients of matmul_i8 (rounding counts as the identity): grad (M,N) = dL/dout in y's type, y
    the layer's output if it ended in a ReLU (its gradient passes where y > 0 or y is -0.0), else None.  -> (grad_x (M,K), grad_weight (N,K), grad_bias (N) fp32),
    None where not wanted.  A factor (gradient times scale) is held to 2^-23 of itself (2^-50 of its row's or column's
    largest where it lies below 2^-27 of that), the sums are fp32, in a fixed order: the same bits every run."""
    _need_gpu(grad)
    M, K = codes.shape
    N = weight_codes.shape[0]
    dev = grad.device
    _i8_device("linear_i8_backward", dev, y, codes, scale, weight_codes, weight_scale)
    if grad.shape != (M, N) or (y is not None and (y.shape != (M, N) or y.dtype != grad.dtype)) \
            or weight_codes.shape[1] != K or scale.shape != (M,) or weight_scale.shape != (N,) \
            or codes.dtype != torch.int8 or weight_codes.dtype != torch.int8 or grad.dtype not in _I8_TYPES \
            or x_dtype not in _I8_TYPES or weight_dtype not in _I8_TYPES:
        raise ValueError("linear_i8_backward: inconsistent shapes or types")
    if M > I8_MAX_K or N > I8_MAX_K or K > I8_MAX_K:
        raise ValueError("linear_i8_backward: (%d, %d, %d); each is at most %d" % (M, N, K, I8_MAX_K))
    if M == 0:
        return (torch.empty((0, K), dtype=x_dtype, device=dev) if want[0] else None,
                torch.zeros((N, K), dtype=weight_dtype, device=dev) if want[1] else None,
                torch.zeros((N,), dtype=torch.float32, device=dev) if want[2] else None)
    codes, weight_codes, scale, weight_scale = _i8_codes(codes), _i8_codes(weight_codes), _f32v(scale), _f32v(weight_scale)
    return _i8_backward(grad, y, codes.data_ptr(), _row_stride(codes), scale.data_ptr(), weight_codes.data_ptr(),
                        _row_stride(weight_codes), weight_scale.data_ptr(), M, N, K, x_dtype, weight_dtype, want)


def _i8_backward(grad, y, codes, codes_stride, scale, weight_codes, weight_stride, weight_scale, M, N, K, x_dtype,
                 weight_dtype, want):
    dev = grad.device
    grad, y = _i8_codes(grad), (_i8_codes(y) if y is not None else None)
    gx = torch.empty((M, K), dtype=x_dtype, device=dev) if want[0] else None
    gw = torch.empty((N, K), dtype=weight_dtype, device=dev) if want[1] else None
    gb = torch.empty((N,), dtype=torch.float32, device=dev) if want[2] else None
    ws, ws_at, nbytes = _i8_workspace("frcnn_linear_i8_backward_workspace_bytes", M, N, K, dev)
    _i8_call("frcnn_linear_i8_backward", dev, grad.data_ptr(), _I8_TYPES[grad.dtype], _row_stride(grad), _at(y),
             _row_stride(y) if y is not None else 0, codes, codes_stride, scale, weight_codes, weight_stride,
             weight_scale, M, N, K, _at(gx), _I8_TYPES[x_dtype], _at(gw), _I8_TYPES[weight_dtype], _at(gb),
             ws_at, nbytes)
    return gx, gw, gb


class FrozenLinearI8(torch.autograd.Function):
    """linear_i8 with the gradient of x (the layer's weights have none): apply(x, weight_codes, weight_scale, bias, relu,
    out_dtype, n_rows).  Rounding of x counts as the identity; rows behind n_rows get zeros."""

    @staticmethod
    def forward(ctx, x, weight_codes, weight_scale, bias=None, relu=False, out_dtype=None, n_rows=None):
        y = linear_i8(x, weight_codes, weight_scale, bias, relu, out_dtype, n_rows)
        ctx.x_dtype = x.dtype
        ctx.save_for_backward(weight_codes, weight_scale, y if relu else None, n_rows)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        codes, scale, y, n_rows = ctx.saved_tensors
        M, (N, K) = grad.shape[0], codes.shape
        if N > I8_MAX_K:
            raise ValueError("FrozenLinearI8: a gradient of %d channels; at most %d" % (N, I8_MAX_K))
        if n_rows is not None:
            grad = grad.where(torch.arange(M, device=grad.device)[:, None] < n_rows, 0)
        codes, scale = _i8_codes(codes), _f32v(scale)
        x_dtype = ctx.x_dtype if ctx.x_dtype in _I8_TYPES else torch.float32
        parts = [grad.new_empty((0, K), dtype=x_dtype)] if M == 0 else []
        for m in range(0, M, I8_MAX_K):  # a row's gradient is its own: as many rows a call as it takes
            g, z = grad[m:m + I8_MAX_K], y[m:m + I8_MAX_K] if y is not None else None
            parts.append(_i8_backward(g, z, None, 0, None, codes.data_ptr(), _row_stride(codes), scale.data_ptr(),
                                      g.shape[0], N, K, x_dtype, torch.float32, (True, False, False))[0])
        gx = parts[0] if len(parts) == 1 else torch.cat(parts)
        return (gx.to(ctx.x_dtype),) + (None,) * 6


@functools.lru_cache(maxsize=1024)
def _i8_saved(M, N, K):
    """Offsets of what frcnn_linear_i8_train leaves for the backward call: x's scales, the weights' codes and scales."""
    ld = (K + 15) // 16 * 16
    up = lambda v: (v + 255) // 256 * 256  # noqa: E731
    x_scale = up(M * ld)
    w = x_scale + up(M * 4)
    return ld, x_scale, w, w + up(N * ld)


class LinearI8(torch.autograd.Function):
    """A dense layer trained through 8-bit rounding: apply(x (M,K), weight (N,K), bias (N) or None, relu) -> (M,N) in
    x's type.  Both operands are quantised by rows on every call (the weights change from step to step), the product
    runs on the codes, and the gradients are linear_i8_backward's."""

    @staticmethod
    def forward(ctx, x, weight, bias=None, relu=False):
        _need_gpu(x, weight, bias)
        if x.dim() != 2 or weight.dim() != 2 or x.shape[1] != weight.shape[1] or weight.shape[0] == 0:
            raise ValueError("LinearI8 expects x (M,K) and weight (N,K); got %s, %s"
                             % (tuple(x.shape), tuple(weight.shape)))
        if x.dtype not in _I8_TYPES or weight.dtype not in _I8_TYPES:
            raise ValueError("LinearI8 takes float32, bfloat16 and float16; got %s, %s" % (x.dtype, weight.dtype))
        dev = x.device
        _i8_device("LinearI8", dev, weight, bias)
        M, K = x.shape
        N = weight.shape[0]
        if K == 0 or K > I8_MAX_K or N > I8_MAX_K or M > I8_MAX_K:
            raise ValueError("LinearI8: (%d, %d, %d); each is at most %d and K at least 1" % (M, N, K, I8_MAX_K))
        if bias is not None and bias.shape != (N,):
            raise ValueError("LinearI8 expects a bias for each of the %d outputs; got %s" % (N, tuple(bias.shape)))
        ctx.relu = relu = bool(relu)
        ctx.types = (x.dtype, weight.dtype, bias.dtype if bias is not None else None)
        ctx.sizes = (M, N, K)
        y = torch.empty((M, N), dtype=x.dtype, device=dev)
        saved = torch.empty((_i8_bytes("frcnn_linear_i8_train_saved_bytes", M, N, K),), dtype=torch.uint8, device=dev)
        if M > 0:
            x, weight, bias = _i8_rows(x, "LinearI8"), _i8_rows(weight, "LinearI8"), _f32v(bias)
            ws, ws_at, nbytes = _i8_workspace("frcnn_linear_i8_train_workspace_bytes", M, N, K, dev)
            _i8_call("frcnn_linear_i8_train", dev, x.data_ptr(), _I8_TYPES[x.dtype], _row_stride(x), weight.data_ptr(),
                     _I8_TYPES[weight.dtype], _row_stride(weight), _at(bias), 1 if relu else 0, M, N, K, y.data_ptr(),
                     _I8_TYPES[y.dtype], N, saved.data_ptr(), saved.numel(), ws_at, nbytes)
        if relu:
            ctx.save_for_backward(saved, y)
        else:
            ctx.save_for_backward(saved)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        saved = ctx.saved_tensors
        M, N, K = ctx.sizes
        x_dtype, w_dtype, b_dtype = ctx.types
        want = (tuple(ctx.needs_input_grad) + (False,))[:3]
        if M == 0:
            return (grad.new_empty((0, K), dtype=x_dtype) if want[0] else None,
                    grad.new_zeros((N, K), dtype=w_dtype) if want[1] else None,
                    grad.new_zeros((N,), dtype=b_dtype) if want[2] else None, None)
        ld, x_scale, w, w_scale = _i8_saved(M, N, K)
        at = saved[0].data_ptr()
        gx, gw, gb = _i8_backward(grad, saved[1] if ctx.relu else None, at, ld, at + x_scale, at + w, ld, at + w_scale,
                                  M, N, K, x_dtype, w_dtype, want)
        if gb is not None and gb.dtype != b_dtype:
            gb = gb.to(b_dtype)
        return gx, gw, gb, None
