"""Torch-facing wrappers over the C ABI of liblmi_hip.so.

PyTorch is plumbing here (device memory, streams); every computation below happens in the HIP
kernels of `csrc/`.  All functions enqueue on the current torch stream and do not synchronise
unless they say so.  There is no CPU fallback: tensors must live on a HIP device.
"""
from __future__ import annotations

import ctypes as C
import functools
import math
import struct
import threading
from typing import List, Optional, Sequence, Tuple, Union

import numpy as np
import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import LMI_F16, LMI_F32, LMI_U8, check, lmi_frame

_L = _lib.load()


class _WorkspaceCache:
    """One growing byte buffer per (device, stream, tag): the library itself never allocates.  At most `limit` buffers
    are held, the least recently used one is dropped first (a process that keeps creating streams would otherwise pin
    one workspace per stream handle it ever used; a dropped buffer goes back to torch's allocator, which orders its
    reuse after the work enqueued on the stream it was allocated on)."""

    def __init__(self, limit: int = 32):
        self._buf = {}
        self._limit = limit
        self._lock = threading.Lock()       # host threads that drive their own streams share this cache

    def get(self, device: torch.device, tag: str, nbytes: int) -> torch.Tensor:
        key = (device.index, torch.cuda.current_stream(device).cuda_stream, tag)
        with self._lock:
            t = self._buf.pop(key, None)
            if t is None or t.numel() < nbytes:
                t = torch.empty((max(nbytes, 256),), dtype=torch.uint8, device=device)
            self._buf[key] = t              # most recently used last (dicts keep insertion order)
            while len(self._buf) > self._limit:
                self._buf.pop(next(iter(self._buf)))
        return t


_ws = _WorkspaceCache()


class _DescriptorCache:
    """Device copies of small descriptor arrays, by content.  A serving loop that letterboxes the same frame buffers
    again (same pointers, same geometry) hands over byte-identical descriptors: the upload -- a pageable host-to-device
    copy, ~100 us, more than the kernel -- then happens once.  The first use synchronises its stream so that later calls
    may read the copy from any stream (and from inside a graph capture, where neither a copy nor a wait is allowed)."""

    def __init__(self, limit: int = 16):
        self._d = {}
        self._limit = limit
        self._lock = threading.Lock()

    def get(self, device: torch.device, raw: bytes) -> torch.Tensor:
        key = (device.index, raw)
        with self._lock:
            t = self._d.pop(key, None)
        if t is None:   # uploaded outside the lock (it synchronises a stream); two threads racing for the same new
            t = torch.frombuffer(bytearray(raw), dtype=torch.uint8).to(device)   # content both upload it, the later entry stays
            if not torch.cuda.is_current_stream_capturing():
                torch.cuda.current_stream(device).synchronize()
        with self._lock:
            self._d[key] = t
            while len(self._d) > self._limit:
                self._d.pop(next(iter(self._d)))
        return t


_desc = _DescriptorCache()


def _stream(device=None) -> int:
    """The current torch stream of `device` (the tensors' device, not whatever device happens to be current)."""
    return torch.cuda.current_stream(device).cuda_stream


def _need_cuda(t: torch.Tensor, name: str) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a tensor on the GPU (there is no CPU fallback for this path)")


def _dt(fp16: bool):
    return (torch.float16, LMI_F16) if fp16 else (torch.float32, LMI_F32)


def letterbox_geometry(h: int, w: int, dst_h: int, dst_w: int, stretch: bool = False):
    """(new_w, new_h, pad_l, pad_r, pad_t, pad_b) -- host arithmetic only."""
    out = (C.c_int32 * 6)()
    check(_L.lmi_letterbox_geometry(h, w, dst_h, dst_w, 1 if stretch else 0, out))
    return tuple(int(v) for v in out)


_FRAME_STRUCT = struct.Struct("<Qiiiiiiii")   # lmi_frame: src, h, w, row_stride, new_w, new_h, pad_l, pad_t, reserved
_FRAME_BYTES = _FRAME_STRUCT.size
assert _FRAME_BYTES == C.sizeof(lmi_frame)
_FRAME_PACK = _FRAME_STRUCT.pack_into


@functools.lru_cache(maxsize=4096)
def _cached_geometry(h: int, w: int, dst_h: int, dst_w: int, stretch: bool, torch_mode: bool, fit):
    """Letterbox geometry of one frame size (a batch usually holds few distinct sizes)."""
    if torch_mode:
        return torch_letterbox_geometry(h, w, dst_h, dst_w, fit)
    return letterbox_geometry(h, w, dst_h, dst_w, stretch)


def preprocess_u8(im: torch.Tensor, fp16: bool = False) -> torch.Tensor:
    """`Yolov8.preprocess` for one uint8 image (H,W) / (H,W,1) / (H,W,3) -> (1,3,H,W)."""
    _need_cuda(im, "im")
    if im.dtype != torch.uint8:
        raise TypeError("preprocess_u8 expects uint8")
    if im.ndim == 2:
        im = im.unsqueeze(-1)
    h, w, c = im.shape
    if im.stride(2) != 1 or im.stride(1) != c:
        im = im.contiguous()
    tdt, ldt = _dt(fp16)
    out = torch.empty((1, 3, h, w), dtype=tdt, device=im.device)
    check(_L.lmi_preprocess_u8(im.data_ptr(), h, w, c, im.stride(0), out.data_ptr(), ldt, _stream(im.device)))
    return out


def torch_letterbox_geometry(h: int, w: int, dst_h: int, dst_w: int, resize=None):
    """(new_w, new_h, pad_l, pad_r, pad_t, pad_b) of the reference helpers' chain `resize_image(im, H=, W=)` then
    `fit_im_to_size(im, H=dst_h, W=dst_w)` (lmi_utils/gadget_utils/pipeline_utils.py:36-39, :110-131): a missing
    side keeps the aspect ratio with `int()`; pads are centred with the smaller half first, negative = centred crop.
    resize = (H, W) as the v1 runner's `--resize h w`; None = the aspect-preserving fit into (dst_h, dst_w)."""
    rh, rw = (None, None) if resize is None else resize
    if rh is None and rw is None:
        if dst_h * w <= dst_w * h:
            rh = dst_h
        else:
            rw = dst_w
    new_w = int(rw) if rw is not None else int(w * rh / h)
    new_h = int(rh) if rh is not None else int(h * rw / w)

    def split(have, want):
        if want >= have:
            before = (want - have) // 2
            return before, want - have - before
        before = (have - want) // 2
        return -before, -(have - want - before)

    pl, pr = split(new_w, dst_w)
    pt, pb = split(new_h, dst_h)
    return new_w, new_h, pl, pr, pt, pb


def _check_lb_out(out, b, dst_h, dst_w, tdt, dev) -> None:
    if not isinstance(out, torch.Tensor) or tuple(out.shape) != (b, 3, dst_h, dst_w) or out.dtype != tdt or not out.is_contiguous() or out.device != dev:
        raise ValueError(f"letterbox: `out` must be a contiguous {tdt} tensor of shape {(b, 3, dst_h, dst_w)} on the frames' device")


def letterbox_tables(frame_hw: Tuple[int, int], dst_hw: Tuple[int, int], device, stretch: bool = False) -> torch.Tensor:
    """Plan half of the uniform cv2-flavoured letterbox (LMI_LB_TABLES_ONLY): the coefficient tables of one geometry
    -- every frame (h, w), destination dst_hw -- built once on the current stream into a buffer the CALLER owns.  Hand it
    to `letterbox(..., tables=t)` and every such call is one launch instead of two; the tables depend on the sizes
    alone (not on pixels, channel order, pad value or dtype), so one buffer serves every call of that geometry, from any
    stream that is ordered after this call, and inside HIP graphs (the buffer must outlive them)."""
    h, w = int(frame_hw[0]), int(frame_hw[1])
    dst_h, dst_w = int(dst_hw[0]), int(dst_hw[1])
    device = torch.device(device)
    if device.type != "cuda":
        raise TypeError("letterbox_tables: the tables live on the GPU (there is no CPU fallback for this path)")
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    t = torch.empty((int(_L.lmi_letterbox_workspace_bytes(1, dst_h, dst_w)),), dtype=torch.uint8, device=device)
    check(_L.lmi_letterbox_u8_uniform(None, 1, h, w, 3 * w, 3 * w * h, None, dst_h, dst_w, LMI_F32, 0, 0, int(stretch),
                                      _lib.LMI_LB_TABLES_ONLY, t.data_ptr(), t.numel(), _stream(device)))
    t._lmi_tables_key = (h, w, dst_h, dst_w, bool(stretch), device.index)
    return t


def letterbox(frames: Union[torch.Tensor, Sequence[torch.Tensor]], dst_hw: Tuple[int, int], pad_value: int = 114,
              swap_rb: bool = False, fp16: bool = False, stretch: bool = False,
              out: Optional[torch.Tensor] = None, mode: str = "cv2", resize=None, torch_threads: Optional[int] = None,
              tables: Optional[torch.Tensor] = None):
    """Fused resize + centred pad + channel swap + /255 + NCHW.

    frames: a (B,H,W,3) uint8 tensor (uniform batch) or a sequence of (H,W,3) uint8 tensors of any
    sizes; grey planes go in as (B,H,W,1) / (H,W) / (H,W,1): they are resampled once and written to the three output
    planes, which is what the callers' GRAY2BGR + resize gives (run_model.py:77-78).  Returns (tensor (B,3,dst_h,dst_w), operators) where operators[b] is the list
    `[{'resize': [new_w,new_h,w,h]}, {'pad': [L,R,T,B]}]` that `revert_to_origin` consumes.
    mode 'cv2': cv2.resize INTER_LINEAR (the callers' default chain); mode 'torch': the reference helpers
    `resize_image` + `fit_im_to_size` (fp32 bilinear, truncating cast; `resize=(H, W)` as the v1 runner's
    `--resize`, either side None; pads may be negative = centred crop; pad value 0 is the helpers' default).
    torch_threads=1 reproduces what those helpers give when torch runs on exactly one thread (aten then picks
    its other CPU kernel for 3-channel frames); any other value: the >= 2-thread result.
    tables: what `letterbox_tables` returned for this geometry (uniform (B,H,W,C) batches, mode 'cv2'): the table pass
    is left out of the call (LMI_LB_TABLES_READY).
    """
    dst_h, dst_w = int(dst_hw[0]), int(dst_hw[1])
    tdt, ldt = _dt(fp16)
    if mode not in ("cv2", "torch"):
        raise ValueError(f"letterbox: unknown mode {mode!r}")
    if resize is not None and mode != "torch":
        raise ValueError("letterbox: resize= belongs to mode='torch' (the cv2 flavour derives its geometry from dst_hw)")
    if isinstance(frames, torch.Tensor):
        if frames.ndim == 2:
            frames = frames[None, :, :, None]
        elif frames.ndim == 3:
            frames = frames.unsqueeze(0)
    if mode == "torch" and isinstance(frames, torch.Tensor):
        frames = list(frames.unbind(0))   # geometry by the helpers' rules: the descriptor form carries it
    if isinstance(frames, torch.Tensor):
        _need_cuda(frames, "frames")
        if frames.dtype != torch.uint8 or frames.ndim != 4 or frames.shape[-1] not in (1, 3):
            raise TypeError("letterbox expects uint8 (B,H,W,3) or, for grey planes, (B,H,W,1)")
        ch = int(frames.shape[-1])
        if frames.stride(3) != 1 or frames.stride(2) != ch:   # frames may start at any byte and lie any distance apart
            frames = frames.contiguous()
        b, h, w, _ = frames.shape
        if out is None:
            out = torch.empty((b, 3, dst_h, dst_w), dtype=tdt, device=frames.device)
        else:
            _check_lb_out(out, b, dst_h, dst_w, tdt, frames.device)
        flags = _lib.LMI_SRC_GRAY if ch == 1 else 0
        if tables is not None:
            if getattr(tables, "_lmi_tables_key", None) != (h, w, dst_h, dst_w, bool(stretch), frames.device.index):
                raise ValueError("letterbox: `tables` were not built by letterbox_tables for this geometry and device")
            ws, flags = tables, flags | _lib.LMI_LB_TABLES_READY
        else:
            ws = _ws.get(frames.device, "letterbox", int(_L.lmi_letterbox_workspace_bytes(1, dst_h, dst_w)))
        check(_L.lmi_letterbox_u8_uniform(frames.data_ptr(), b, h, w, frames.stride(1), frames.stride(0), out.data_ptr(),
                                          dst_h, dst_w, ldt, pad_value, int(swap_rb), int(stretch), flags, ws.data_ptr(),
                                          ws.numel(), _stream(frames.device)))
        g = letterbox_geometry(h, w, dst_h, dst_w, stretch)
        ops = [[{"resize": [g[0], g[1], w, h]}, {"pad": [g[2], g[3], g[4], g[5]]}] for _ in range(b)]
        return out, ops
    if tables is not None:
        raise ValueError("letterbox: tables= serves uniform (B,H,W,C) batches in mode 'cv2'")
    frames = list(frames)
    if not frames:
        raise ValueError("letterbox: empty batch")
    # the per-frame work below is host time on the caller's critical path (64 frames: 235 us before, more than the
    # kernels): geometry from a cache keyed by the frame size, descriptors packed straight into one byte buffer
    keep = []
    nf = len(frames)
    raw = bytearray(_FRAME_BYTES * nf)
    ops = []
    ch = None
    fit = (dst_h, dst_w) if stretch else resize
    fit = None if fit is None else (fit[0], fit[1])
    for i, f in enumerate(frames):
        if not isinstance(f, torch.Tensor) or not f.is_cuda:
            _need_cuda(f, f"frames[{i}]")
        if f.ndim == 2:
            f = f.unsqueeze(-1)
        if f.dtype != torch.uint8 or f.ndim != 3 or f.shape[-1] not in (1, 3):
            raise TypeError("letterbox expects uint8 (H,W,3) frames, or grey planes (H,W) / (H,W,1)")
        h, w, c = f.shape
        if ch is None:
            ch = int(c)
        elif c != ch:
            raise ValueError("letterbox: one batch holds either colour frames or grey planes, not both")
        s0, s1, s2 = f.stride()
        if s2 != 1 or s1 != ch:
            f = f.contiguous()
            s0 = f.stride(0)
        keep.append(f)
        g = _cached_geometry(h, w, dst_h, dst_w, stretch, mode == "torch", fit)
        _FRAME_PACK(raw, _FRAME_BYTES * i, f.data_ptr(), h, w, s0, g[0], g[1], g[2], g[4], 0)
        ops.append([{"resize": [g[0], g[1], w, h]}, {"pad": [g[2], g[3], g[4], g[5]]}])
    desc = (C.c_char * len(raw)).from_buffer(raw)   # the host copy the C ABI validates (lmi_frame[nf], same layout)
    dev = keep[0].device
    ddev = _desc.get(dev, bytes(raw))
    if out is None:
        out = torch.empty((len(keep), 3, dst_h, dst_w), dtype=tdt, device=dev)
    else:
        _check_lb_out(out, len(keep), dst_h, dst_w, tdt, dev)
    ws = _ws.get(dev, "letterbox", int(_L.lmi_letterbox_workspace_bytes(len(keep), dst_h, dst_w)))
    check(_L.lmi_letterbox_u8(C.addressof(desc), ddev.data_ptr(), len(keep), out.data_ptr(), dst_h, dst_w, ldt,
                              pad_value, int(swap_rb), ((2 if torch_threads == 1 else 1) if mode == "torch" else 0) | (_lib.LMI_SRC_GRAY if ch == 1 else 0),
                              ws.data_ptr(), ws.numel(), _stream(dev)))
    ddev.record_stream(torch.cuda.current_stream(dev))
    return out, ops


def _finalize_setup(b: int, max_det: int, nc: int, dev, model_hw, orig_hw, thres, pad_round: bool, with_slots: bool, out, kpt=None):
    """Buffers + the lmi_finalize_args record shared by finalize_detections and the fused nms_v8(finalize=...).
    Returns (result dict, args struct, tensors to keep alive until the call is enqueued)."""
    if out is not None:   # reuse a previous result dict of the same shapes
        keep, keep_count = out["keep"], out["keep_count"]
        mask_slot, slot_map, slot_base = out["mask_slot"], out["slot_map"], out["slot_base"]
        if keep.shape != (b, max_det) or keep.dtype != torch.uint8 or keep.device != dev or not keep.is_contiguous():
            raise ValueError("finalize: `out` buffers do not match this call's shapes")
    else:
        keep = torch.empty((b, max_det), dtype=torch.uint8, device=dev)
        keep_count = torch.empty((b,), dtype=torch.int32, device=dev)
        mask_slot = torch.empty((b, max_det), dtype=torch.int32, device=dev) if with_slots else None
        slot_map = torch.empty((b * max_det,), dtype=torch.int32, device=dev) if with_slots else None
        slot_base = torch.empty((b + 1,), dtype=torch.int32, device=dev) if with_slots else None
    alive = []
    if isinstance(orig_hw, torch.Tensor):
        _need_cuda(orig_hw, "orig_hw")
        ohw = orig_hw.to(torch.int32).contiguous()
        if ohw.shape != (b, 2):
            raise ValueError("orig_hw must be (B,2)")
        alive.append(ohw)
        ohw_ptr, uh, uw = ohw.data_ptr(), 0, 0
    else:
        ohw_ptr, uh, uw = None, int(orig_hw[0]), int(orig_hw[1])
    if isinstance(thres, torch.Tensor):
        _need_cuda(thres, "thres")
        th = thres.to(torch.float64).contiguous()
        if th.numel() != nc:
            raise ValueError("per-class thresholds must have nc entries")
        alive.append(th)
        th_ptr, ut = th.data_ptr(), 0.0
    else:
        th_ptr, ut = None, float(thres)
    p = lambda t: t.data_ptr() if t is not None else None
    args = _lib.lmi_finalize_args(int(model_hw[0]), int(model_hw[1]), uh, uw, ohw_ptr, int(bool(pad_round)), 0, th_ptr, ut,
                                  keep.data_ptr(), keep_count.data_ptr(), p(mask_slot), p(slot_map), p(slot_base),
                                  *((int(kpt[0]), int(kpt[1]), int(kpt[2]), 0) if kpt else (0, 0, 0, 0)))
    res = {"keep": keep, "keep_count": keep_count, "mask_slot": mask_slot, "slot_map": slot_map, "slot_base": slot_base}
    return res, args, alive


def nms_v8(pred: torch.Tensor, conf_thres: float, iou_thres: float = 0.45, agnostic: bool = False, max_det: int = 300,
           nc: int = 0, max_nms: int = 30000, max_wh: float = 7680.0, out=None, rotated: bool = False,
           decode_done: Optional[torch.cuda.Event] = None, finalize: Optional[dict] = None, sweep_only: bool = False):
    """`ops.non_max_suppression` on the head output (B, 4+nc+nm, A), fp32 or fp16 (an fp16 head is read as it is,
    every value promoted to fp32 in the kernels: the result of `pred.float()` without that pass).  rotated=True:
    oriented boxes (xywh + angle as the last extra channel, ultralytics' nms_rotated on probiou), rows stay xywh.
    decode_done: an event recorded on the current stream between the candidate filter (HBM-bound) and the
    sort + suppression pass (latency-bound): work on another stream that waits for it shares the chip with the
    latter (lmi_nms_decode_ex / lmi_nms_suppress_ex instead of the one-call lmi_nms_v8_ex; same result).
    finalize: dict(model_hw=, orig_hw=, thres=[, pad_round=True, with_slots=True, out=None, kpt=(col0, nkpt, ndim)]) -- kpt:
    keypoint models, `scale_coords` on those row columns in the same launch (`Yolov8Pose.postprocess`); otherwise the arguments of
    finalize_detections: scale_boxes + clip, class threshold and survivor ranks then run in the suppression kernel's
    epilogue (one launch less, same results) and the call returns a 4th value, finalize_detections' result dict.

    sweep_only: LMI_NMS_SWEEP_ONLY -- keep the one-workgroup sorted sweep where the suppressor-list kernel would run
    first (same result; measurement and tests).

    Returns (det (B,max_det,6+nm) fp32, count (B,) int32, anchor (B,max_det) int32), all on the
    device; rows >= count[b] are unspecified.  `out` = a previous result tuple of the same shapes
    to write into instead of allocating (serving loops)."""
    _need_cuda(pred, "pred")
    if pred.dtype not in (torch.float32, torch.float16):
        pred = pred.float()
    if not pred.is_contiguous():
        pred = pred.contiguous()
    pdt = LMI_F16 if pred.dtype == torch.float16 else LMI_F32
    b, ch, a = pred.shape
    nc = nc or (ch - 4)
    nm = ch - nc - 4
    if nm < 0:
        raise ValueError(f"nc={nc} does not fit a head with {ch} channels")
    dev = pred.device
    if out is not None:
        det, count, anchor = out
        if det.shape != (b, max_det, 6 + nm) or count.shape != (b,) or anchor.shape != (b, max_det):
            raise ValueError("nms_v8: `out` buffers do not match this call's shapes")
        if det.dtype != torch.float32 or count.dtype != torch.int32 or anchor.dtype != torch.int32:
            raise ValueError("nms_v8: `out` buffers must be (float32, int32, int32)")
        if not (det.is_contiguous() and count.is_contiguous() and anchor.is_contiguous()) or det.device != dev:
            raise ValueError("nms_v8: `out` buffers must be contiguous and on the head's device")
    else:
        det = torch.empty((b, max_det, 6 + nm), dtype=torch.float32, device=dev)
        count = torch.empty((b,), dtype=torch.int32, device=dev)
        anchor = torch.empty((b, max_det), dtype=torch.int32, device=dev)
    fin_res, fin_ptr, alive = None, None, None
    if finalize is not None:
        if rotated:
            raise ValueError("nms_v8: finalize= serves axis-aligned boxes (use finalize_obb for rotated ones)")
        fin_res, fin_args, alive = _finalize_setup(b, max_det, nc, dev, finalize["model_hw"], finalize["orig_hw"], finalize["thres"],
                                                   finalize.get("pad_round", True), finalize.get("with_slots", True), finalize.get("out"),
                                                   finalize.get("kpt"))
        fin_ptr = C.addressof(fin_args)
    nbytes = int(_L.lmi_nms_workspace_bytes(b, a))
    ws = _ws.get(dev, "nms", nbytes)
    st = _stream(dev)
    if decode_done is not None:
        check(_L.lmi_nms_decode_ex(pred.data_ptr(), pdt, b, nc, nm, a, float(conf_thres), ws.data_ptr(), ws.numel(), st))
        decode_done.record()
        check(_L.lmi_nms_suppress_ex(pred.data_ptr(), pdt, b, nc, nm, a, float(iou_thres), int(agnostic), int(max_det), int(max_nms),
                                     float(max_wh), int(rotated) | (_lib.LMI_NMS_SWEEP_ONLY if sweep_only else 0), fin_ptr, det.data_ptr(),
                                     count.data_ptr(), anchor.data_ptr(), ws.data_ptr(), ws.numel(), st))
    else:
        check(_L.lmi_nms_v8_ex(pred.data_ptr(), pdt, b, nc, nm, a, float(conf_thres), float(iou_thres), int(agnostic), int(max_det),
                               int(max_nms), float(max_wh), int(rotated) | (_lib.LMI_NMS_SWEEP_ONLY if sweep_only else 0), fin_ptr, det.data_ptr(),
                               count.data_ptr(), anchor.data_ptr(), ws.data_ptr(), ws.numel(), st))
    if finalize is not None:
        return det, count, anchor, fin_res
    return det, count, anchor


def finalize_obb(det: torch.Tensor, count: torch.Tensor, nc: int, model_hw: Tuple[int, int],
                 orig_hw: Union[Tuple[int, int], torch.Tensor], thres: Union[float, torch.Tensor]):
    """regularize_rboxes + scale_boxes(xywh=True) + xywhr2xyxyxyxy + per-class threshold on rotated NMS rows.
    Returns dict(corners (B,max_det,4,2) fp32, keep (B,max_det) uint8, keep_count (B,)); det is not modified."""
    _need_cuda(det, "det")
    b, max_det, stride = det.shape
    dev = det.device
    corners = torch.empty((b, max_det, 4, 2), dtype=torch.float32, device=dev)
    keep = torch.empty((b, max_det), dtype=torch.uint8, device=dev)
    keep_count = torch.empty((b,), dtype=torch.int32, device=dev)
    if isinstance(orig_hw, torch.Tensor):
        _need_cuda(orig_hw, "orig_hw")
        ohw = orig_hw.to(torch.int32).contiguous()
        ohw_ptr, uh, uw = ohw.data_ptr(), 0, 0
    else:
        ohw_ptr, uh, uw = None, int(orig_hw[0]), int(orig_hw[1])
    if isinstance(thres, torch.Tensor):
        _need_cuda(thres, "thres")
        th = thres.to(torch.float64).contiguous()
        if th.numel() != nc:
            raise ValueError("per-class thresholds must have nc entries")
        th_ptr, ut = th.data_ptr(), 0.0
    else:
        th_ptr, ut = None, float(thres)
    check(_L.lmi_finalize_obb(det.data_ptr(), count.data_ptr(), b, max_det, stride, nc, int(model_hw[0]), int(model_hw[1]),
                              ohw_ptr, uh, uw, th_ptr, ut, corners.data_ptr(), keep.data_ptr(), keep_count.data_ptr(), _stream(det.device)))
    return {"corners": corners, "keep": keep, "keep_count": keep_count}


def finalize_detections(det: torch.Tensor, count: torch.Tensor, nc: int, model_hw: Tuple[int, int],
                        orig_hw: Union[Tuple[int, int], torch.Tensor], thres: Union[float, torch.Tensor],
                        pad_round: bool = True, with_slots: bool = True, out=None):
    """scale_boxes + clip IN PLACE on det[..., :4], per-class threshold, dense survivor ranks.

    orig_hw: (H0, W0) for every image, or an int32 device tensor (B,2).  thres: a float, or a
    float64 device tensor (nc,) of per-class thresholds.
    Returns dict(keep (B,max_det) uint8, keep_count (B,), mask_slot, slot_map, slot_base (B+1,))."""
    _need_cuda(det, "det")
    if det.dtype != torch.float32 or not det.is_contiguous() or det.ndim != 3:
        raise ValueError("finalize_detections: det must be a contiguous float32 (B,max_det,6+nm) tensor")
    b, max_det, stride = det.shape
    res, a, alive = _finalize_setup(b, max_det, nc, det.device, model_hw, orig_hw, thres, pad_round, with_slots, out)
    check(_L.lmi_finalize_detections(det.data_ptr(), count.data_ptr(), b, max_det, stride, nc, a.model_h, a.model_w, a.orig_hw,
                                     a.uniform_h0, a.uniform_w0, a.pad_round, a.thres, a.uniform_thres, a.keep, a.keep_count,
                                     a.mask_slot, a.slot_map, a.slot_base, _stream(det.device)))
    return res


def scale_coords(det: torch.Tensor, count: torch.Tensor, nkpt: int, ndim: int, model_hw: Tuple[int, int],
                 orig_hw: Union[Tuple[int, int], torch.Tensor], col0: int = 6) -> torch.Tensor:
    """`ops.scale_coords` IN PLACE on the keypoint columns det[..., col0 : col0 + nkpt*ndim] of the NMS rows."""
    _need_cuda(det, "det")
    b, max_det, stride = det.shape
    if isinstance(orig_hw, torch.Tensor):
        _need_cuda(orig_hw, "orig_hw")
        ohw = orig_hw.to(torch.int32).contiguous()
        ohw_ptr, uh, uw = ohw.data_ptr(), 0, 0
    else:
        ohw_ptr, uh, uw = None, int(orig_hw[0]), int(orig_hw[1])
    check(_L.lmi_scale_coords(det.data_ptr(), count.data_ptr(), b, max_det, stride, int(col0), int(nkpt), int(ndim),
                              int(model_hw[0]), int(model_hw[1]), ohw_ptr, uh, uw, _stream(det.device)))
    return det


_MASK_DTYPES = {torch.uint8: LMI_U8, torch.bool: LMI_U8, torch.float32: LMI_F32}


def _mask_flags(logits: str, upsample: str) -> int:
    if logits not in ("rows", "mfma") or upsample not in ("split", "single"):
        raise ValueError("process_mask: logits must be 'rows' | 'mfma', upsample 'split' | 'single'")
    return (_lib.LMI_MASK_LOGITS_MFMA if logits == "mfma" else 0) | (_lib.LMI_MASK_UPSAMPLE_SINGLE if upsample == "single" else 0)


def _check_window(mh: int, mw: int, h0: int, w0: int) -> None:
    """ultralytics' scale_masks crops the letterbox pad off the prototype window before interpolating; for an extremely
    thin frame that window is empty and F.interpolate raises -- same exception type and wording here."""
    gain = min(mh / h0, mw / w0)
    pad_x, pad_y = (mw - w0 * gain) / 2, (mh - h0 * gain) / 2
    wh_, ww_ = int(mh - pad_y) - int(pad_y), int(mw - pad_x) - int(pad_x)
    if wh_ <= 0 or ww_ <= 0:
        raise RuntimeError(f"Input and output sizes should be greater than 0, but got input (H: {max(wh_, 0)}, W: {max(ww_, 0)}) "
                           f"output (H: {h0}, W: {w0})")


def _mask_inputs(proto, det, slot_map, slot_base, logits="rows"):
    """Validated inputs -> (prototypes, flag).  The prototypes of an fp16 model (`fp16=True`) are read as they are
    (LMI_MASK_PROTO_F16: promoted to fp32 in the kernel = `protos.float()` without that pass) whenever the row kernel
    serves the shape; any other dtype is converted first."""
    _need_cuda(proto, "proto")
    half = proto.dtype == torch.float16 and logits == "rows" and proto.ndim == 4 and proto.shape[-1] % 2 == 0
    if proto.dtype != torch.float32 and not half:
        proto = proto.float()
    if not proto.is_contiguous():
        proto = proto.contiguous()
    for t, name, dt in ((det, "det", torch.float32), (slot_map, "slot_map", torch.int32), (slot_base, "slot_base", torch.int32)):
        _need_cuda(t, name)
        if t.dtype != dt or not t.is_contiguous() or t.device != proto.device:
            raise ValueError(f"process_mask: {name} must be a contiguous {dt} tensor on the prototypes' device")
    if det.ndim != 3 or det.shape[0] != proto.shape[0] or slot_base.numel() != proto.shape[0] + 1:
        raise ValueError("process_mask: det must be (B,max_det,6+nm) and slot_base (B+1,)")
    return proto, (_lib.LMI_MASK_PROTO_F16 if half else 0)


def process_mask(proto: torch.Tensor, det: torch.Tensor, slot_map: torch.Tensor, slot_base: torch.Tensor,
                 orig_hw: Tuple[int, int], capacity: int, out_dtype: torch.dtype = torch.uint8,
                 out: Optional[torch.Tensor] = None, split_events=None, before_upsample=None, logits: str = "rows",
                 upsample: str = "split"):
    """`process_mask_native` + `masks[M]` for the whole batch (uniform original size).

    Returns (masks (capacity,H0,W0) of uint8|float32 in slot order, overflow (1,) int32).
    split_events: optional (start, end) torch.cuda.Event pair recorded around the upsample stage
    alone (the two halves are then enqueued through lmi_mask_logits / lmi_mask_upsample).
    before_upsample: optional callable run between the two halves (e.g. joining another stream: nothing should run
    beside the upsample's zero fill, see profiles/r01/write_ceiling.md).
    logits='mfma' / upsample='single' select the dense MFMA product / the one-pass upsample kernel (measurement)."""
    proto, pflag = _mask_inputs(proto, det, slot_map, slot_base, logits)
    b, nm, mh, mw = proto.shape
    _, max_det, stride = det.shape
    h0, w0 = int(orig_hw[0]), int(orig_hw[1])
    _check_window(mh, mw, h0, w0)
    ldt = _MASK_DTYPES[out_dtype]   # torch.bool: the kernels' 0/1 bytes ARE bools (same storage as uint8)
    capacity = max(int(capacity), 1)
    if out is None:
        out = torch.empty((capacity, h0, w0), dtype=out_dtype, device=proto.device)
    elif tuple(out.shape) != (capacity, h0, w0) or out.dtype != out_dtype or not out.is_contiguous() or out.device != proto.device:
        raise ValueError(f"process_mask: `out` must be a contiguous {out_dtype} tensor of shape {(capacity, h0, w0)} on the prototypes' device")
    overflow = torch.empty((1,), dtype=torch.int32, device=proto.device)
    nbytes = int(_L.lmi_mask_workspace_bytes(capacity, mh, mw))
    ws = _ws.get(proto.device, "mask", nbytes)
    flags, st = _mask_flags(logits, upsample) | pflag, _stream(proto.device)
    if split_events is None and before_upsample is None:
        check(_L.lmi_process_mask_ex(proto.data_ptr(), b, nm, mh, mw, det.data_ptr(), max_det, stride, slot_map.data_ptr(),
                                     slot_base.data_ptr(), h0, w0, None, None, out.data_ptr(), ldt, capacity, 0, overflow.data_ptr(),
                                     ws.data_ptr(), ws.numel(), flags, st))
    else:
        check(_L.lmi_mask_logits_ex(proto.data_ptr(), b, nm, mh, mw, det.data_ptr(), max_det, stride, slot_map.data_ptr(),
                                    slot_base.data_ptr(), h0, w0, None, None, capacity, ws.data_ptr(), ws.numel(), flags, st))
        if before_upsample is not None:
            before_upsample()
        if split_events is not None:
            split_events[0].record()
        check(_L.lmi_mask_upsample_ex(ws.data_ptr(), b, nm, mh, mw, det.data_ptr(), max_det, stride, slot_map.data_ptr(),
                                      slot_base.data_ptr(), h0, w0, None, None, out.data_ptr(), ldt, capacity, 0, overflow.data_ptr(),
                                      flags, _stream(proto.device)))
        if split_events is not None:
            split_events[1].record()
    return out, overflow


def process_mask_ragged(proto: torch.Tensor, det: torch.Tensor, slot_map: torch.Tensor, slot_base: torch.Tensor,
                        sizes: Sequence[Tuple[int, int]], counts: Sequence[int], out_dtype: torch.dtype = torch.uint8,
                        logits: str = "rows", upsample: str = "split") -> List[torch.Tensor]:
    """`process_mask_native` + `masks[M]` for a batch of DIFFERENTLY sized originals in one launch (the reference loops
    over the images, object_detectors/yolov8_lmi/model.py:215-236).  sizes[b] = (H0, W0); counts[b] = survivors of
    image b as read from slot_base (the caller synchronised to size its outputs anyway).  The masks are packed into
    one flat buffer, every image's block starting on a 16-element boundary; returns the per-image views
    [(counts[b], H0_b, W0_b)], empty images included."""
    proto, pflag = _mask_inputs(proto, det, slot_map, slot_base, logits)
    b, nm, mh, mw = proto.shape
    _, max_det, stride = det.shape
    if len(sizes) != b or len(counts) != b:
        raise ValueError("process_mask_ragged: one size and one count per image")
    ldt = _MASK_DTYPES[out_dtype]   # torch.bool: the kernels' 0/1 bytes ARE bools (same storage as uint8)
    desc = (_lib.lmi_mask_image * b)()
    off = 0
    for i, ((h0, w0), n) in enumerate(zip(sizes, counts)):
        h0, w0, n = int(h0), int(w0), int(n)
        _check_window(mh, mw, h0, w0)
        desc[i] = _lib.lmi_mask_image(h0, w0, n, 0, off)
        off = (off + n * h0 * w0 + 15) & ~15
    total = int(sum(int(c) for c in counts))
    dev = proto.device
    flat = torch.empty((max(off, 16),), dtype=out_dtype, device=dev)
    views = [flat[d.out_offset:d.out_offset + d.n_masks * d.h0 * d.w0].view(d.n_masks, d.h0, d.w0) for d in desc]
    if total == 0:
        return views
    ddev = torch.frombuffer(bytearray(bytes(desc)), dtype=torch.uint8).to(dev)
    ws = _ws.get(dev, "mask", int(_L.lmi_mask_workspace_bytes(total, mh, mw)))
    st = _stream(dev)
    check(_L.lmi_process_mask_ex(proto.data_ptr(), b, nm, mh, mw, det.data_ptr(), max_det, stride, slot_map.data_ptr(),
                                 slot_base.data_ptr(), 0, 0, C.addressof(desc), ddev.data_ptr(), flat.data_ptr(), ldt, total, flat.numel(),
                                 None, ws.data_ptr(), ws.numel(), _mask_flags(logits, upsample) | pflag, st))
    ddev.record_stream(torch.cuda.current_stream(dev))
    return views


def point_ops(operations: Sequence[dict]):
    """Operator list -> (ctypes array of lmi_point_op, n) for lmi_revert_points_f32.  The divisor of a 'resize'
    is the Python-float ratio rounded to fp32, as `torch.tensor([tw/orig_w, th/orig_h])` does
    (lmi_utils/gadget_utils/pipeline_utils.py:447)."""
    rows = []
    for op in operations:
        if 'resize' in op:
            tw, th, ow, oh = op['resize']
            rows.append((_lib.LMI_POINT_DIV, tw / ow, th / oh))
        elif 'pad' in op:
            rows.append((_lib.LMI_POINT_SUB, op['pad'][0], op['pad'][2]))
        elif 'stretch' in op:
            rows.append((_lib.LMI_POINT_DIV, op['stretch'][0], op['stretch'][1]))
        elif 'flip' in op:
            lr, ud, im_w, im_h = op['flip']
            if lr or ud:
                kind = _lib.LMI_POINT_FLIP_XY if (lr and ud) else (_lib.LMI_POINT_FLIP_X if lr else _lib.LMI_POINT_FLIP_Y)
                rows.append((kind, im_w, im_h))
        else:
            raise Exception(f'unsupported operation: {op}')
    arr = (_lib.lmi_point_op * max(len(rows), 1))()
    for i, (k, x, y) in enumerate(rows):
        arr[i].kind, arr[i].x, arr[i].y = k, float(np.float32(x)), float(np.float32(y))
    return arr, len(rows)


def revert_points(pts: torch.Tensor, operations: Sequence[dict]) -> torch.Tensor:
    """`pipeline_utils.revert_to_origin` for an fp32 (N,2) / (N,4) tensor on the device: one launch for the whole
    array whatever the length of the operator list.  Returns a new tensor."""
    _need_cuda(pts, "pts")
    if pts.ndim != 2 or pts.shape[1] not in (2, 4):
        raise Exception(f'pts should be Nx2 or Nx4, got shape: {pts.shape}')
    if pts.dtype != torch.float32:
        raise TypeError("revert_points handles fp32 points (what the detector emits)")
    src = pts.contiguous()
    out = torch.empty_like(src)
    arr, n = point_ops(operations)
    check(_L.lmi_revert_points_f32(src.data_ptr(), src.numel() // 2, C.cast(arr, C.c_void_p), n, out.data_ptr(), _stream(src.device)))
    return out


def mask_stages(h: int, w: int, operations: Sequence[dict]):
    """Split the reverted operator list into fused stages [(fit_h, fit_w, resize_h, resize_w, lr, ud, out_h, out_w)]:
    every stage is at most one centred crop/pad, then one resize, then one flip, in that order."""
    stages, cur = [], None

    def flush():
        nonlocal cur
        if cur is not None:
            stages.append(cur)
            cur = None

    def need(level):  # 1 fit, 2 resize, 3 flip: a stage applies them in ascending order, once each
        nonlocal cur
        if cur is None or cur["level"] >= level:
            flush()
            cur = {"level": 0, "fit": (0, 0), "resize": (0, 0), "lr": False, "ud": False}
        cur["level"] = level

    for op in reversed(list(operations)):
        if 'resize' in op:
            _, _, ow, oh = op['resize']
            need(2)
            cur["resize"] = (int(oh), int(ow))
            h, w = int(oh), int(ow)
        if 'pad' in op:
            left, right, top, bottom = op['pad']
            nh, nw = h - top - bottom, w - left - right
            if nh <= 0 or nw <= 0:
                raise ValueError(f"pad {op['pad']} leaves no pixels of a {h}x{w} mask")
            need(1)
            cur["fit"] = (int(nh), int(nw))
            h, w = int(nh), int(nw)
        if 'flip' in op:
            lr, ud = bool(op['flip'][0]), bool(op['flip'][1])
            if lr or ud:
                need(3)
                cur["lr"], cur["ud"] = lr, ud
        if cur is not None:
            cur["out"] = (h, w)
    flush()
    return [(s["fit"][0], s["fit"][1], s["resize"][0], s["resize"][1], s["lr"], s["ud"], s["out"][0], s["out"][1]) for s in stages]


def revert_masks(masks: torch.Tensor, operations: Sequence[dict]) -> torch.Tensor:
    """`pipeline_utils.revert_masks_to_origin` for a stack (m,H,W) of fp32 or uint8 masks on the device: one launch
    per fused stage for ALL masks (the reference loops over masks in Python, three torch ops each)."""
    _need_cuda(masks, "masks")
    if masks.ndim != 3:
        raise ValueError(f"masks must be (m,H,W), got {tuple(masks.shape)}")
    ldt = {torch.uint8: LMI_U8, torch.float32: LMI_F32}.get(masks.dtype)
    if ldt is None:
        raise TypeError("revert_masks handles fp32 and uint8 masks")
    cur = masks.contiguous()
    m = cur.shape[0]
    for fit_h, fit_w, rs_h, rs_w, lr, ud, oh, ow in mask_stages(cur.shape[1], cur.shape[2], operations):
        out = torch.empty((m, oh, ow), dtype=cur.dtype, device=cur.device)
        check(_L.lmi_revert_masks_stage(cur.data_ptr(), ldt, m, cur.shape[1], cur.shape[2], fit_h, fit_w, rs_h, rs_w,
                                        1 if lr else 0, 1 if ud else 0, out.data_ptr(), _stream(cur.device)))
        cur = out
    return cur


def paste_masks(masks: torch.Tensor, boxes: torch.Tensor, image_shape: Tuple[int, int], threshold: float = 0.5) -> torch.Tensor:
    """`rescale_masks` (lmi_utils/postprocess_utils/mask_utils.py:66-140): (N,Hm,Wm) soft masks pasted into their xyxy
    boxes of an (H,W) image, `>= threshold`.  Returns a bool tensor (N,H,W) like the reference; for threshold < 0, like
    the reference, the sampled values themselves as uint8 (value * 255, truncated)."""
    _need_cuda(masks, "masks")
    _need_cuda(boxes, "boxes")
    if masks.ndim != 3 or masks.shape[-1] != masks.shape[-2]:
        raise AssertionError("Only square mask predictions are supported")
    n = masks.shape[0]
    if boxes.shape[0] != n:
        raise AssertionError(tuple(boxes.shape))
    h, w = int(image_shape[0]), int(image_shape[1])
    out = torch.empty((n, h, w), dtype=torch.uint8, device=masks.device)
    soft = threshold < 0    # the reference's visualisation mode: (value * 255).to(uint8) instead of a bool mask
    if n == 0:
        return out if soft else out.bool()
    m = masks.float().contiguous()
    b = boxes.float().contiguous()
    check(_L.lmi_paste_masks(m.data_ptr(), n, m.shape[1], m.shape[2], b.data_ptr(), b.shape[1], h, w, float(threshold),
                             out.data_ptr(), _stream(m.device)))
    return out if soft else out.view(torch.bool)


_FLOAT_DTYPES = {torch.float32: LMI_F32, torch.float16: LMI_F16, torch.bfloat16: _lib.LMI_BF16}


def _launch(entry, args, device: torch.device, *more) -> None:
    """entry(args, *more, stream) on the current stream of `device`, which is made the current device for it if it is not."""
    index = device.index
    if index == torch.cuda.current_device():
        status = entry(args, *more, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            status = entry(args, *more, torch._C._cuda_getCurrentRawStream(index))
    if status:
        check(status)


def _not_traced(what: str) -> None:
    """A trace (torch.jit.trace, make_fx) records torch's own operations: of the ones below it would keep the allocation of the result and not the kernel
    that fills it.  Refused.  (torch.compile breaks its graph at the calls below and runs them as they are.)"""
    if torch._C._is_tracing() or (torch._C._len_torch_dispatch_stack() and torch._C._get_dispatch_mode(_PROXY) is not None):
        raise RuntimeError(f"{what} cannot be traced: its kernel would be missing from the graph")


_PROXY = torch._C._TorchDispatchModeKey.PROXY


def _no_gradient(what: str, *tensors) -> None:
    """The operators below serve inference: a graph they would silently cut is refused, and so are tangents of forward mode, and a trace."""
    _not_traced(what)
    if forward_ad._current_level >= 0 and any(isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{what} has no gradient: call it on the primals (torch.autograd.forward_ad.unpack_dual)")
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in tensors):
        raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad() / inference_mode(), or detach its inputs")


_ACTIVATIONS = {"softmax": _lib.LMI_PROB_SOFTMAX, "sigmoid": _lib.LMI_PROB_SIGMOID, "none": _lib.LMI_PROB_NONE}
_LABEL_DTYPES = {torch.float32: LMI_F32, torch.int32: _lib.LMI_I32, torch.int64: _lib.LMI_I64}


def _two_strides(t: torch.Tensor, nd: int):
    """Leading `nd` dimensions of t as (n0, n1, stride0, stride1), or None where two strides cannot say it."""
    n, st = [], []
    for size, stride in zip(t.shape[:nd], t.stride()[:nd]):
        if size == 1:
            continue
        if n and st[-1] == stride * size:      # folds into the dimension before it
            n[-1], st[-1] = n[-1] * size, stride
        else:
            n.append(size)
            st.append(stride)
    if len(n) > 2:
        return None
    while len(n) < 2:
        n.insert(0, 1)
        st.insert(0, 0)
    return n[0], n[1], st[0], st[1]


def class_logprobs(x: torch.Tensor, labels: Optional[torch.Tensor] = None, top: int = 0, activation: str = "softmax",
                   index: Optional[torch.Tensor] = None, count: Optional[torch.Tensor] = None, out: Optional[dict] = None) -> dict:
    """Log probability of given classes, entropy, and the `top` best classes of every row of x (..., C), classes last,
    fp32 / fp16 / bf16.  x is read where it lies: a transposed view of the head's class planes
    (`pred[:, 4:4 + nc].transpose(1, 2)`) or of the distance bins costs no copy.

    activation 'softmax': x are logits, one class per row (a row of -inf alone has log probabilities -inf, entropy 0);
    'sigmoid': logits of independent classes, the entropy summed over the yes / no answers; 'none': such
    probabilities themselves, as the detection head emits them.
    labels (...): int64, int32 or float32 (the class column of NMS rows, `det[:, :, 5]`, as it is); outside [0, C): NaN.
    index (B, M) int32: row (b, m) is read at x[b, index[b, m]] of x (B, A, C) -- `anchor` of nms_v8; labels and results are
    (B, M) then.  count (B,) int32: rows m >= count[b] are skipped and the results there left as they are (unspecified in
    fresh ones).
    out: a previous result of the same shapes to write into instead of allocating; not in the memory of x, labels, index or count.
    Returns dict(logprob (...) if labels are given, entropy (...), and for top > 0 top_logprob, top_index (..., top)): fp32 and int32, best
    first, equal values in class order, NaN first.  Inference only: inputs that require a gradient are refused."""
    _need_cuda(x, "x")
    _no_gradient("class_logprobs", x)
    if x.dtype not in _FLOAT_DTYPES:
        raise TypeError("class_logprobs: x must be float32, float16 or bfloat16")
    act = _ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"class_logprobs: unknown activation {activation!r}")
    if x.ndim < 1 or x.shape[-1] < 1:
        raise ValueError("class_logprobs: x must hold at least one class in its last dimension")
    dev, c, top = x.device, x.shape[-1], int(top)
    if not 0 <= top <= min(c, _lib.LMI_MAX_TOP):
        raise ValueError(f"class_logprobs: top={top} must lie in 0..{min(c, _lib.LMI_MAX_TOP)}")
    lead = tuple(x.shape[:-1])
    if index is not None:
        if x.ndim != 3 or index.ndim != 2 or index.shape[0] != x.shape[0]:
            raise ValueError("class_logprobs: index (B,M) needs x (B,A,C)")
        if index.dtype != torch.int32 or not index.is_contiguous() or index.device != dev:
            raise ValueError("class_logprobs: index must be a contiguous int32 tensor on x's device")
        lead = tuple(index.shape)
    if count is not None:
        if len(lead) != 2 or tuple(count.shape) != lead[:1] or count.dtype != torch.int32 or not count.is_contiguous() or count.device != dev:
            raise ValueError("class_logprobs: count must be a contiguous int32 tensor (B,) on x's device, rows (B,M)")
    if labels is not None:
        if labels.dtype not in _LABEL_DTYPES or labels.device != dev:
            raise TypeError("class_logprobs: labels must be int64, int32 or float32 on x's device")
        if tuple(labels.shape) != lead:
            raise ValueError(f"class_logprobs: labels must have shape {lead}")
    want = [("entropy", lead, torch.float32)]
    if labels is not None:
        want.append(("logprob", lead, torch.float32))
    if top:
        want += [("top_logprob", lead + (top,), torch.float32), ("top_index", lead + (top,), torch.int32)]
    res = {}
    for key, size, dtype in want:
        if out is None:
            res[key] = torch.empty(size, dtype=dtype, device=dev)
            continue
        t = res[key] = out.get(key)
        if t is None or t.shape != size or t.dtype != dtype or t.device != dev or not t.is_contiguous():
            raise ValueError(f"class_logprobs: out[{key!r}] must be a contiguous {dtype} tensor of shape {size} on x's device")
    out = res
    rows = math.prod(lead)
    if rows == 0:
        return out
    if index is not None or count is not None:   # the two leading dimensions mean what they say
        if x.ndim != 3:
            raise ValueError("class_logprobs: count needs x (B,M,C)")
        n0, n1, s0, s1 = lead[0], lead[1], x.stride(0), x.stride(1)
    else:
        split = _two_strides(x, x.ndim - 1)
        if split is None:
            x = x.contiguous()
            split = _two_strides(x, x.ndim - 1)
        n0, n1, s0, s1 = split
    cs = x.stride(-1) if c > 1 else 1
    if cs == 0 or any(v < 0 for v in (s0, s1, cs)):   # classes broadcast from one value
        x = x.contiguous()
        n0, n1, s0, s1 = (n0, n1, x.stride(0), x.stride(1)) if x.ndim == 3 and (index is not None or count is not None) else _two_strides(x, x.ndim - 1)
        cs = x.stride(-1)
    l0 = l1 = 0
    if labels is not None:
        if (n0, n1) == lead:
            l0, l1 = labels.stride()
        else:
            if not labels.is_contiguous():
                labels = labels.contiguous()
            l0, l1 = n1, 1
    workspace, need = None, 0
    if c >= _lib.LMI_LOGPROB_SPLIT_FROM:
        need = int(_L.lmi_class_logprobs_workspace_bytes(n0 * n1, c, cs, _FLOAT_DTYPES[x.dtype]))
        if need:   # not from the shared cache: two captured graphs that run side by side must not share it
            workspace = torch.empty((need,), dtype=torch.uint8, device=dev)
    args = _lib.LOGPROB_ARGS.pack(
        x.data_ptr(), _FLOAT_DTYPES[x.dtype], act, c, cs, n0, n1, s0, s1, 0 if index is None else index.data_ptr(),
        0 if index is None else x.shape[1], 0 if count is None else count.data_ptr(), 0 if labels is None else labels.data_ptr(), l0, l1,
        0 if labels is None else _LABEL_DTYPES[labels.dtype], top, 0 if labels is None else out["logprob"].data_ptr(), out["entropy"].data_ptr(),
        out["top_logprob"].data_ptr() if top else 0, out["top_index"].data_ptr() if top else 0, workspace.data_ptr() if need else 0, need)
    _launch(_L.lmi_class_logprobs, args, dev)   # refuses results over an input or one another, from the addresses it has at hand
    return out


def _mx_sizes(shape):
    """Shapes of an MxTensor's parts: ((S, G, 1024), (Q, G, 256))."""
    groups = -(-math.prod(shape[:-1]) // 32)
    steps = -(-shape[-1] // 64)
    return (steps, groups, 1024), (-(-steps // 4), groups, 256)


class MxTensor:
    """A tensor (..., k) in MXFP4: blocks of 32 elements along the last dimension share a power-of-two scale; 4.25 bits per
    element.  The blocks lie in the order the matrix instruction takes them, k in steps of 64 (two blocks), rows in groups of
    32: packed uint8 (S, G, 1024), a group's kilobyte as (block, row, 16 bytes), two elements per byte, the earlier one in
    the low half; scales uint8 (Q, G, 256), the bytes of four steps as (block, row, step): 2^(byte - 127), 255 = NaN.
    G = ceil(rows / 32), S = ceil(k / 64), Q = ceil(S / 4); what lies beyond the tensor is zero."""

    __slots__ = ("packed", "scales", "shape")

    def __init__(self, packed: torch.Tensor, scales: torch.Tensor, shape):
        self.packed, self.scales, self.shape = packed, scales, torch.Size(shape)
        if len(self.shape) < 1 or self.shape[-1] < 1:
            raise ValueError("MxTensor: shape must end in at least one element")
        for t, s, name in zip((packed, scales), _mx_sizes(self.shape), ("packed", "scales")):
            if t.dtype != torch.uint8 or tuple(t.shape) != s or not t.is_contiguous() or t.device != packed.device:
                raise ValueError(f"MxTensor: {name} must be a contiguous uint8 tensor of shape {s} on one device with the other")

    @property
    def device(self) -> torch.device:
        return self.packed.device

    def __repr__(self):
        return f"MxTensor(shape={tuple(self.shape)}, device={self.device})"


def _rows_of(x: torch.Tensor):
    """x (..., k) as (tensor, rows, row stride): the elements of a row side by side, rows a fixed distance apart."""
    if x.ndim == 1:
        x = x.unsqueeze(0)
    if x.shape[-1] > 1 and x.stride(-1) != 1:
        x = x.contiguous()
    split = _two_strides(x, x.ndim - 1)
    if split is None or split[0] != 1:
        x = x.contiguous()
        split = _two_strides(x, x.ndim - 1)
    return x, math.prod(x.shape[:-1]), split[3]


def mx_quantize(x: torch.Tensor) -> MxTensor:
    """x (..., k), fp32 / fp16 / bf16 -> MXFP4 along the last dimension: scale 2^(floor(log2 max|x|) - 2) of each block of 32, elements
    rounded to nearest (ties to even) and held at 6 at most.  A block with an infinity or a NaN becomes NaN as a whole."""
    _need_cuda(x, "x")
    _no_gradient("mx_quantize", x)
    if x.dtype not in _FLOAT_DTYPES:
        raise TypeError("mx_quantize: x must be float32, float16 or bfloat16")
    if x.ndim < 1 or x.shape[-1] < 1:
        raise ValueError("mx_quantize: x must hold at least one element in its last dimension")
    shape, k, dev = x.shape, x.shape[-1], x.device
    size_p, size_s = _mx_sizes(shape)
    q = MxTensor.__new__(MxTensor)
    packed = q.packed = torch.empty(size_p, dtype=torch.uint8, device=dev)
    scales = q.scales = torch.empty(size_s, dtype=torch.uint8, device=dev)
    q.shape = shape
    rows = x.numel() // k
    if rows:
        if x.is_contiguous():
            stride = k
        else:
            x, _, stride = _rows_of(x)
        _launch(_L.lmi_mx_quantize, x.data_ptr(), dev, _FLOAT_DTYPES[x.dtype], rows, k, stride, packed.data_ptr(), scales.data_ptr())
    return q


def _need_mx(q, name: str) -> None:
    if not isinstance(q, MxTensor):
        raise TypeError(f"{name} must be an MxTensor (mx_quantize)")
    _need_cuda(q.packed, name)


def mx_dequantize(q: MxTensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values an MxTensor stands for (exact in fp32 and, within its range, bf16; fp16 rounds what lies outside its range)."""
    _need_mx(q, "q")
    _not_traced("mx_dequantize")
    if dtype not in _FLOAT_DTYPES:
        raise TypeError("mx_dequantize: dtype must be float32, float16 or bfloat16")
    y = torch.empty(q.shape, dtype=dtype, device=q.device)
    if y.numel():
        _launch(_L.lmi_mx_dequantize, q.packed.data_ptr(), q.device, q.scales.data_ptr(), math.prod(q.shape[:-1]), q.shape[-1], y.data_ptr(),
                _FLOAT_DTYPES[dtype])
    return y


_MX_ACTS = {None: _lib.LMI_ACT_NONE, "silu": _lib.LMI_ACT_SILU}


def _mx_product(what, x_ptr, x_scales, x_dtype, batch, pixels, k, x_batch, x_stride, weight, bias, act, y, layout):
    """Checks what mx_linear and mx_pointwise share, and enqueues the product."""
    dev = y.device
    if bias is not None and (bias.dtype != torch.float32 or tuple(bias.shape) != (weight.shape[0],) or not bias.is_contiguous() or bias.device != dev):
        raise ValueError(f"{what}: bias must be a contiguous float32 tensor ({weight.shape[0]},) on x's device")
    if y.numel() == 0:
        return y
    fields = [x_ptr, x_scales or 0, x_dtype, _MX_ACTS[act], batch, pixels, k, weight.shape[0], x_batch, x_stride, weight.packed.data_ptr(),
              weight.scales.data_ptr(), 0 if bias is None else bias.data_ptr(), y.data_ptr(), _FLOAT_DTYPES[y.dtype], layout, 0, 0]
    args = _lib.MX_PRODUCT_ARGS.pack(*fields)
    need = int(_L.lmi_mx_product_workspace_bytes(args))
    if need:   # not from the shared cache: two captured graphs that run side by side must not share it
        workspace = torch.empty((need,), dtype=torch.uint8, device=dev)
        fields[-2:] = workspace.data_ptr(), need
        args = _lib.MX_PRODUCT_ARGS.pack(*fields)
    _launch(_L.lmi_mx_product, args, dev)
    return y


def _mx_common(what, x, weight, bias, act, k):
    _need_mx(weight, "weight")
    _no_gradient(what, x, bias)
    if len(weight.shape) != 2 or weight.shape[1] != k or weight.shape[0] < 1:
        raise ValueError(f"{what}: weight {tuple(weight.shape)} does not fit inputs of {k} channels (out, in)")
    if weight.device != x.device:
        raise ValueError(f"{what}: weight must be on x's device")
    if act not in _MX_ACTS:
        raise ValueError(f"{what}: unknown activation {act!r} (None or 'silu')")


def _span(t: torch.Tensor):
    """First byte of t and the one behind its last (t not empty)."""
    first = t.data_ptr()
    if t.is_contiguous():
        return first, first + t.nbytes
    return first, first + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))


def _apart(what: str, out: torch.Tensor, inputs: dict) -> None:
    """Refuses a result that lies in the memory of an input (None and empty tensors lie nowhere)."""
    first, last = _span(out)
    for name, t in inputs.items():
        if t is not None and t.numel():
            a, b = _span(t)
            if first < b and a < last:
                raise ValueError(f"{what}: `out` lies in the memory of {name}")


def _mx_out(what, out, x, weight, bias, shape, dtype, memory_format=torch.contiguous_format):
    if out is None:
        return torch.empty(shape, dtype=dtype, device=x.device, memory_format=memory_format)
    if tuple(out.shape) != tuple(shape) or out.dtype != dtype or out.device != x.device or not out.is_contiguous(memory_format=memory_format):
        raise ValueError(f"{what}: `out` must be a {dtype} tensor of shape {tuple(shape)} in {memory_format} on x's device")
    if out.numel():   # every result needs whole rows of x and of the weights, which others overwrite by then
        parts = {"x": x.packed, "x's scales": x.scales} if isinstance(x, MxTensor) else {"x": x}
        _apart(what, out, {**parts, "weight": weight.packed, "weight's scales": weight.scales, "bias": bias})
    return out


def mx_linear(x: Union[torch.Tensor, MxTensor], weight: MxTensor, bias: Optional[torch.Tensor] = None, act: Optional[str] = None,
              dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """act(x weight^T + bias) with both factors in MXFP4 and fp32 sums: x (..., k) is quantised as `mx_quantize` does it, on the
    fly, or comes quantised (MxTensor); weight MxTensor (n, k); bias fp32 (n,); act None | 'silu'.
    dtype: of the result, x's own (which it must be if given) or, for an MxTensor, float32 unless said otherwise.
    out: a tensor to write into, not in the memory of x, weight or bias.  Inference only."""
    quantised = isinstance(x, MxTensor)
    if quantised:
        _need_mx(x, "x")
        dtype = dtype or torch.float32
        if dtype not in _FLOAT_DTYPES:
            raise TypeError("mx_linear: dtype must be float32, float16 or bfloat16")
    else:
        _need_cuda(x, "x")
        if x.dtype not in _FLOAT_DTYPES:
            raise TypeError("mx_linear: x must be float32, float16, bfloat16 or an MxTensor")
        if dtype not in (None, x.dtype):
            raise ValueError("mx_linear: the result has x's dtype unless x is an MxTensor")
        dtype = x.dtype
    if not len(x.shape):
        raise ValueError("mx_linear: x must be (..., k)")
    k = x.shape[-1]
    _mx_common("mx_linear", x.packed if quantised else x, weight, bias, act, k)
    y = _mx_out("mx_linear", out, x, weight, bias, tuple(x.shape[:-1]) + (weight.shape[0],), dtype)
    m = math.prod(x.shape[:-1])
    if quantised:
        return _mx_product("mx_linear", x.packed.data_ptr(), x.scales.data_ptr(), _lib.LMI_MXFP4, 1, m, k, 0, 0, weight, bias, act, y, _lib.LMI_MX_ROWS)
    stride = k
    if m and not x.is_contiguous():
        x, _, stride = _rows_of(x)
        if stride >= 1 << 24:
            x = x.contiguous()
            stride = k
    return _mx_product("mx_linear", x.data_ptr(), None, _FLOAT_DTYPES[dtype], 1, m, k, 0, stride, weight, bias, act, y, _lib.LMI_MX_ROWS)


def mx_pointwise(x: torch.Tensor, weight: MxTensor, bias: Optional[torch.Tensor] = None, act: Optional[str] = None,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """A 1x1 convolution in MXFP4: x (B, k, H, W) fp32 / fp16 / bf16, quantised on the fly in blocks of 32 channels of a pixel,
    weight MxTensor (n, k), bias fp32 (n,), act None | 'silu', fp32 sums.  Returns (B, n, H, W) of x's dtype, channels-last
    if x is.  Channel slices of a larger map (`chunk` along dim 1) are read in place.  out: a tensor to write into, not in the memory of x,
    weight or bias.  Inference only."""
    _need_cuda(x, "x")
    if x.dtype not in _FLOAT_DTYPES:
        raise TypeError("mx_pointwise: x must be float32, float16 or bfloat16")
    if x.ndim != 4:
        raise ValueError("mx_pointwise: x must be (B, k, H, W)")
    b, k, h, w = x.shape
    _mx_common("mx_pointwise", x, weight, bias, act, k)
    n = weight.shape[0]
    sb, sk, sh, sw = x.stride()
    if b == 1:        # strides of dimensions of one element say nothing, however large or odd
        sb = 0
    if k == 1:
        sk = 0
    planes = (w == 1 or sw == 1) and (h == 1 or sh == w * (sw if w > 1 else 1)) and h * w > 1
    if planes and w == 1 and h > 1:
        planes = sh == 1
    rows = (k == 1 or sk == 1) and not planes and (h == 1 or w == 1 or sh == w * sw)
    step = sk if planes else sb if h * w == 1 else sw if w > 1 else sh   # between neighbouring channels or rows
    if (not planes and not rows) or step >= 1 << 24:
        x = x.contiguous()
        sb, sk, sh, sw = k * h * w, h * w, w, 1
        planes = h * w > 1
    if planes:
        y = _mx_out("mx_pointwise", out, x, weight, bias, (b, n, h, w), x.dtype)
        return _mx_product("mx_pointwise", x.data_ptr(), None, _FLOAT_DTYPES[x.dtype], b, h * w, k, sb, sk, weight, bias, act, y, _lib.LMI_MX_PLANES)
    fmt = torch.channels_last if h * w > 1 else torch.contiguous_format   # one pixel: both are the same memory
    y = _mx_out("mx_pointwise", out, x, weight, bias, (b, n, h, w), x.dtype, fmt)
    if h * w == 1:       # an image per row
        return _mx_product("mx_pointwise", x.data_ptr(), None, _FLOAT_DTYPES[x.dtype], 1, b, k, 0, sb, weight, bias, act, y, _lib.LMI_MX_ROWS)
    return _mx_product("mx_pointwise", x.data_ptr(), None, _FLOAT_DTYPES[x.dtype], b, h * w, k, sb, sw if w > 1 else sh, weight, bias, act, y,
                       _lib.LMI_MX_ROWS)
