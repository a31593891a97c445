"""The networks' forward with and without MXFP4 1x1 convolutions: fp16, random weights, 640 x 640, both memory layouts, batch norms as
they are and folded into the convolutions; ms, medians of blocks taken in turn."""
import copy
import os
import sys

import torch
from torch.nn.utils.fusion import fuse_conv_bn_eval

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from object_detectors_amd.nets.yolov8 import ConvBNAct, YoloV8  # noqa: E402


def folded(m):
    for q in m.modules():
        if isinstance(q, ConvBNAct):
            q.conv, q.bn = fuse_conv_bn_eval(q.conv, q.bn), torch.nn.Identity()
    return m


def block(f, n):
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    torch.cuda.synchronize()
    a.record()
    for _ in range(n):
        f()
    b.record()
    torch.cuda.synchronize()
    return a.elapsed_time(b) / n


for scale in ("n", "s", "x"):
    for batch in (1, 16):
        for layout in ("planes", "channels-last"):
            torch.manual_seed(0)
            base = YoloV8(scale, 80, True).eval().cuda().half()
            x = torch.rand(batch, 3, 640, 640, device="cuda", dtype=torch.half)
            if layout == "channels-last":
                base, x = base.to(memory_format=torch.channels_last), x.contiguous(memory_format=torch.channels_last)
            mx = copy.deepcopy(base)
            mx.quantize_pointwise()
            nets = {"fp16": base, "fp16 folded": folded(copy.deepcopy(base)), "mx": mx, "mx folded": folded(copy.deepcopy(mx))}
            times = {k: [] for k in nets}
            with torch.inference_mode():
                for m in nets.values():
                    block(lambda: m(x), 3)
                for _ in range(7):
                    for k, m in nets.items():
                        times[k].append(block(lambda: m(x), 5))
            print(scale, "batch", batch, layout + ":", ", ".join(f"{k} {sorted(t)[3]:.2f}" for k, t in times.items()), flush=True)
