"""The operators as they are used together: a network whose 1x1 convolutions run in MXFP4, its head through NMS, and the
evidence of the kept detections in the results -- every stage against its oracle on the values that really passed."""
import os
import sys

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DROPIN = os.path.join(ROOT, "object_detectors_amd", "dropin")
if DROPIN not in sys.path:
    sys.path.insert(0, DROPIN)

from oracle import boxes as OB, class_logprobs as OC, mx as OM, nms as ON  # noqa: E402
from object_detectors_amd import synth  # noqa: E402
from object_detectors_amd.nets.yolov8 import ConvBNAct, MxPointwise, YoloV8  # noqa: E402

NAMES = {0: "person", 1: "car", 2: "dog", 3: "cat"}


def _net(task, seed=7):
    torch.manual_seed(seed)
    m = YoloV8("n", 4, names=NAMES, task=task)
    for conv in m.head.cv3:
        conv[-1].bias.data.normal_(-2.0, 0.5)
        conv[-1].weight.data.mul_(8.0)
    for mod in m.modules():            # batch norms with something to fold
        if isinstance(mod, torch.nn.BatchNorm2d):
            mod.running_mean.normal_(0, 0.1)
            mod.running_var.uniform_(0.5, 1.5)
    return m.eval()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("channels_last", [False, True])
def test_every_layer_of_a_forward(dtype, channels_last):
    """Each replaced convolution, on the activations of a real forward, against the oracle's product of the folded weights."""
    ref = _net("segment").cuda()
    net = _net("segment").cuda()
    if dtype == torch.float16:
        net.half()
    folded = {}
    for name, m in ref.named_modules():
        if isinstance(m, ConvBNAct) and m.conv.kernel_size == (1, 1):
            gain = (m.bn.weight / torch.sqrt(m.bn.running_var + m.bn.eps)).detach()
            folded[name] = (m.conv.weight.detach().flatten(1) * gain[:, None], m.bn.bias.detach() - m.bn.running_mean * gain)
    n = net.quantize_pointwise()
    mods = {name: m for name, m in net.named_modules() if isinstance(m, MxPointwise)}
    assert len(mods) == n and set(mods) == {k for k in folded if not k.startswith("head")} and n > 15
    seen = {}
    hooks = [m.register_forward_hook(lambda m, a, y, name=name: seen.update({name: (a[0], y)})) for name, m in mods.items()]
    x = torch.rand(2, 3, 96, 160, device="cuda", dtype=dtype)
    if channels_last:
        x = x.contiguous(memory_format=torch.channels_last)
        net = net.to(memory_format=torch.channels_last)
    with torch.inference_mode():
        net(x)
    for h in hooks:
        h.remove()
    assert set(seen) == set(mods)
    for name, (a, y) in seen.items():
        w, b = folded[name]
        k = w.shape[1]
        xr = a.permute(0, 2, 3, 1).reshape(-1, k).double().cpu().numpy()
        # the weights the layer holds: an fp16 network folds its rounded weights
        m = mods[name]
        packed, scales, _ = OM.rows_of(m.packed.cpu().numpy(), m.scales.cpu().numpy(), w.shape[0], k)
        wq = OM.dequantize(OM.unpack(packed), scales, k)
        if dtype == torch.float32:
            assert np.array_equal(wq, OM.values(w.double().cpu().numpy()))
        xq = OM.values(xr)
        bias = m.bias.double().cpu().numpy()
        assert np.abs(bias - b.double().cpu().numpy()).max() <= (2e-3 if dtype == torch.float16 else 1e-6)
        want, size = xq @ wq.T + bias, np.abs(xq) @ np.abs(wq).T + np.abs(bias)
        want = want / (1 + np.exp(-want))
        # fp32 sums of k terms (2^-23 each), SiLU's slope 1.1 and 8 units of its own, one rounding to the type
        tol = (k + 8) * 2.0 ** -23 * size * 1.1 + np.abs(want) * (8 * 2.0 ** -24 + torch.finfo(dtype).eps / 2) * 1.01 + 6e-8
        got = y.permute(0, 2, 3, 1).reshape(-1, w.shape[0]).double().cpu().numpy()
        assert (np.abs(got - want) <= tol).all(), name


def test_the_head_too():
    """head=True takes the head's 1x1 layers as well, those without norm and activation included; a second call finds none."""
    net = _net("segment").cuda()
    plain = {name: (m.weight.detach().flatten(1).clone(), m.bias.detach().clone()) for name, m in net.named_modules()
             if isinstance(m, torch.nn.Conv2d) and m.kernel_size == (1, 1) and m.bias is not None}
    few = sum(isinstance(m, torch.nn.Conv2d) and m.kernel_size == (1, 1) for m in net.modules())
    assert net.quantize_pointwise(head=True) == few and net.quantize_pointwise(head=True) == 0
    mods = {name: m for name, m in net.named_modules() if isinstance(m, MxPointwise)}
    assert len(plain) == 9 and set(plain) < set(mods)
    seen = {}
    for name in plain:
        mods[name].register_forward_hook(lambda m, a, y, name=name: seen.update({name: (a[0], y)}))
    with torch.inference_mode():
        net(torch.rand(2, 3, 96, 160, device="cuda"))
    for name, (w, b) in plain.items():
        a, y = seen[name]
        want, size = OM.product(a.permute(0, 2, 3, 1).reshape(-1, w.shape[1]).double().cpu().numpy(), w.double().cpu().numpy(), b.double().cpu().numpy())
        got = y.permute(0, 2, 3, 1).reshape(-1, w.shape[0]).double().cpu().numpy()
        assert (np.abs(got - want) <= (w.shape[1] + 8) * 2.0 ** -23 * size + 1e-37).all(), name


@pytest.mark.parametrize("task", ["detect", "segment", "pose", "obb"])
@pytest.mark.parametrize("fp16", [False, True])
def test_predict_with_evidence(tmp_path, task, fp16):
    from object_detectors_amd.wrapper import Yolov8Core, Yolov8ObbCore, Yolov8PoseCore
    import _paths  # noqa: F401
    base = {"detect": Yolov8Core, "segment": Yolov8Core, "pose": Yolov8PoseCore, "obb": Yolov8ObbCore}[task]

    class Model(base):
        mx_weights = True
        alternatives = 3

    m = _net(task)
    path = str(tmp_path / "w.pt")
    torch.save({"format": "lmi-yolov8-torch", "scale": "n", "nc": 4, "seg": task == "segment", "task": task, "names": NAMES,
                "kpt_shape": [17, 3], "state_dict": m.state_dict()}, path)
    model = Model.__new__(Model)
    model._init(path, fp16=fp16)
    assert any(isinstance(q, MxPointwise) for q in model.model.modules())
    image = synth.frames_u8(np.random.default_rng(5), 1, 320, 320)[0]
    plain = Model.__new__(Model)
    plain._init(path, fp16=fp16)
    plain.alternatives = 0
    for tensor in (False, True):
        im = torch.from_numpy(image).cuda() if tensor else image
        # one forward for every side: the library's convolutions need not give the same bits twice
        with torch.inference_mode():
            pred = type(model).forward(model, model.preprocess(im))
        head = (pred[0] if isinstance(pred, (tuple, list)) else pred).float().cpu().numpy()
        model.forward = plain.forward = lambda _im: pred
        r, _ = model.predict(im, 0.2)
        q, _ = plain.predict(im, 0.2)
        assert set(r) - set(q) == {"logprobs", "entropy", "alternatives"}          # what was there before is as it was
        same = lambda a, b: np.array_equal(np.asarray(a.cpu() if isinstance(a, torch.Tensor) else a), np.asarray(b.cpu() if isinstance(b, torch.Tensor) else b))
        assert same(r["boxes"], q["boxes"]) and same(r["scores"], q["scores"]) and r["classes"] == q["classes"]
        n = len(r["scores"])
        assert n > 3 and len(r["logprobs"]) == len(r["entropy"]) == len(r["alternatives"]) == n
        assert isinstance(r["entropy"], torch.Tensor if tensor else np.ndarray)
        scores = np.asarray(r["scores"].cpu() if tensor else r["scores"])
        rows = head[0, 4:8].T
        lp = np.asarray(r["logprobs"].cpu() if tensor else r["logprobs"])
        ent = np.asarray(r["entropy"].cpu() if tensor else r["entropy"])
        assert np.allclose(lp, np.log(scores.astype(np.float64)), rtol=1e-6, atol=1e-7)
        for i in range(n):        # the detection's anchor: the one whose best class has this score (and whose row gives these results)
            hits = np.nonzero(rows.max(1) == scores[i])[0]
            ref = OC.evidence(rows[hits], None, 3, "none")
            ok = [j for j in range(len(hits)) if [NAMES[c] for c in ref["top_index"][j]] == [a[0] for a in r["alternatives"][i]]
                  and np.allclose(ref["top_logprob"][j], [a[1] for a in r["alternatives"][i]], rtol=1e-6, atol=1e-7)
                  and abs(ref["entropy"][j] - ent[i]) <= 1e-5 * max(1.0, ref["entropy"][j])]
            assert ok and r["alternatives"][i][0][0] == r["classes"][i]


def test_batch_results_line_up(tmp_path):
    """predict_batch: an image without detections adds no entry, the others' evidence belongs to their own rows."""
    from object_detectors_amd.wrapper import Yolov8Core
    m = _net("detect")
    path = str(tmp_path / "w.pt")
    torch.save({"format": "lmi-yolov8-torch", "scale": "n", "nc": 4, "seg": False, "names": NAMES, "state_dict": m.state_dict()}, path)
    model = Yolov8Core.__new__(Yolov8Core)
    model._init(path)
    model.alternatives = 9                     # more than there are classes: all of them
    rng = np.random.default_rng(0)
    B, S = 3, 320
    head = synth.head(rng, B, 4, 0, S, objects=12)
    head[1, 4:] = 0.0                          # nothing in the second image
    frames = [np.zeros((S, S, 3), np.uint8)] * B
    img = torch.zeros(B, 3, S, S)
    r = model.postprocess(torch.from_numpy(head).cuda(), img, frames, 0.3, _with_index=True)
    assert r["image_index"] == [0, 2] and len(r["entropy"]) == len(r["alternatives"]) == 2
    ref = ON.non_max_suppression(head, 0.3, 0.45, nc=4)
    for j, i in enumerate((0, 2)):
        rd, ra = ref[i]
        M = OB.class_filter(rd[:, 4], rd[:, 5], np.full(4, 0.3))
        want = OC.evidence(head[i, 4:].T[ra][M], rd[M, 5].astype(int), 4, "none")
        assert np.allclose(r["logprobs"][j], want["logprob"], rtol=1e-6, atol=1e-7)
        assert np.allclose(r["entropy"][j], want["entropy"], rtol=1e-5)
        assert [[NAMES[c] for c in row] for row in want["top_index"]] == [[a[0] for a in row] for row in r["alternatives"][j]]
