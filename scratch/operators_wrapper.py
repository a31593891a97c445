"""What `alternatives` costs in the wrapper: postprocess of 64 images of 300 kept rows, 80 classes, numpy and tensor frames; ms, medians."""
import os
import sys
import time

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from object_detectors_amd import synth  # noqa: E402
from object_detectors_amd.wrapper import Yolov8Core  # noqa: E402

B, S = 64, 640
head = torch.from_numpy(synth.head(np.random.default_rng(0), B, 80, 0, S, objects=400)).cuda()
model = Yolov8Core.__new__(Yolov8Core)
model.device, model._thres_cache = torch.device("cuda:0"), {}
model.model = type("Net", (), {"names": {i: f"class{i}" for i in range(80)}, "fp16": False})()
img = torch.zeros(B, 3, S, S)
for kind in ("numpy", "tensor"):
    frame = np.zeros((S, S, 3), np.uint8)
    frames = [frame if kind == "numpy" else torch.from_numpy(frame).cuda()] * B
    for k in (0, 5):
        model.alternatives = k
        times = []
        for _ in range(12):
            torch.cuda.synchronize()
            t0 = time.perf_counter()
            r = model.postprocess(head, img, frames, 0.05, return_segments=False)
            torch.cuda.synchronize()
            times.append((time.perf_counter() - t0) * 1e3)
        print(f"{kind} frames, alternatives {k}: {sorted(times)[6]:.2f} ms, {sum(len(c) for c in r['classes'])} rows", flush=True)
