"""Refusals of class_logprobs and the MXFP4 operators that need no GPU, and the oracles against hand-made values."""
import ctypes as C

import numpy as np
import pytest
import torch

from oracle import class_logprobs as OC, mx as OM


@pytest.fixture(scope="module")
def L():
    from object_detectors_amd import _lib
    return _lib


def test_cpu_tensors_are_refused():
    from object_detectors_amd import hip_ops as ops
    from object_detectors_amd.nets.yolov8 import YoloV8
    with pytest.raises(TypeError, match="GPU"):
        ops.class_logprobs(torch.zeros(2, 3))
    with pytest.raises(TypeError, match="GPU"):
        ops.mx_quantize(torch.zeros(2, 32))
    q = ops.MxTensor(torch.zeros(1, 1, 1024, dtype=torch.uint8), torch.zeros(1, 1, 256, dtype=torch.uint8), (2, 30))
    with pytest.raises(TypeError, match="GPU"):
        ops.mx_dequantize(q)
    with pytest.raises(TypeError, match="GPU"):
        ops.mx_linear(torch.zeros(1, 30), q)
    with pytest.raises(TypeError, match="GPU"):
        ops.mx_pointwise(torch.zeros(1, 30, 2, 2), q)
    with pytest.raises(RuntimeError, match="eval"):
        YoloV8("n", 2).quantize_pointwise()
    with pytest.raises(TypeError, match="GPU"):
        YoloV8("n", 2).eval().quantize_pointwise()


@pytest.mark.parametrize("packed,scales,shape", [((2, 32), (2, 2), (2, 33)), ((1, 1, 1024), (1, 1, 256), (33, 33)),
                                                 ((1, 1, 1024), (1, 1, 256), (2, 65)), ((2, 1, 1024), (2, 1, 256), (2, 65)),
                                                 ((5, 1, 1024), (1, 1, 256), (2, 300))])
def test_mx_tensor_checks_its_parts(packed, scales, shape):
    from object_detectors_amd import hip_ops as ops
    with pytest.raises(ValueError, match="MxTensor"):
        ops.MxTensor(torch.zeros(packed, dtype=torch.uint8), torch.zeros(scales, dtype=torch.uint8), shape)


def _probs(L, **kw):
    a = L.lmi_logprob_args()
    a.x, a.x_dtype, a.activation, a.classes, a.class_stride, a.n0, a.n1, a.stride0, a.stride1 = 4096, 0, 0, 10, 1, 1, 4, 40, 10
    for k, v in kw.items():
        setattr(a, k, v)
    return L.load().lmi_class_logprobs(C.byref(a), None)


def test_class_logprobs_arguments(L):
    lib = L.load()
    assert lib.lmi_class_logprobs(None, None) == -1
    assert _probs(L, n1=0) == 0                      # no rows: nothing to do, nothing is read
    for bad in (dict(classes=0), dict(n0=-1), dict(activation=3), dict(top=-1), dict(top=11), dict(top=33, classes=100), dict(x=None),
                dict(x_dtype=2), dict(class_stride=0), dict(stride1=-1), dict(labels=4096, label_dtype=2), dict(index=4096)):
        assert _probs(L, **bad) == -1, bad
    assert _probs(L, classes=1 << 31) == -4 and _probs(L, n0=1 << 20, n1=1 << 12) == -4
    need = lib.lmi_class_logprobs_workspace_bytes(2, 200001, 1, 0)
    assert need > 0 and lib.lmi_class_logprobs_workspace_bytes(2, 80, 1, 0) == 0
    assert _probs(L, classes=200001, n1=2) == -3
    assert _probs(L, classes=200001, n1=2, workspace=4096, workspace_bytes=need - 1) == -3
    assert _probs(L, classes=200001, n1=2, workspace=4104, workspace_bytes=need) == -2


def _product(L, **kw):
    a = L.lmi_mx_product_args()
    a.x, a.x_dtype, a.act, a.batch, a.pixels, a.k, a.n, a.x_stride = 4096, 0, 0, 1, 4, 64, 8, 64
    a.w_packed, a.w_scales, a.y, a.y_dtype = 4096, 4096, 4096, 0
    for k, v in kw.items():
        setattr(a, k, v)
    return L.load().lmi_mx_product(C.byref(a), None)


def test_mx_arguments(L):
    lib = L.load()
    assert lib.lmi_mx_quantize(4096, 0, 0, 32, 32, 4096, 4096, None) == 0 and lib.lmi_mx_dequantize(4096, 4096, 0, 32, 4096, 0, None) == 0
    for bad in ((None, 0, 1, 32, 32, 4096, 4096), (4096, 2, 1, 32, 32, 4096, 4096), (4096, 0, -1, 32, 32, 4096, 4096), (4096, 0, 1, 0, 32, 4096, 4096),
                (4096, 0, 1, 32, 32, None, 4096)):
        assert lib.lmi_mx_quantize(*bad, None) == -1, bad
    assert lib.lmi_mx_quantize(4096, 0, 1, 32, 32, 4104, 4096, None) == -2
    assert lib.lmi_mx_quantize(4096, 0, 1 << 41, 32, 32, 4096, 4096, None) == -4
    assert lib.lmi_mx_dequantize(4096, 4096, 1, 32, 4096, 2, None) == -1 and lib.lmi_mx_dequantize(4096, None, 1, 32, 4096, 0, None) == -1
    assert lib.lmi_mx_product(None, None) == -1
    assert _product(L, pixels=0) == 0
    for bad in (dict(k=0), dict(n=0), dict(batch=-1), dict(act=2), dict(x_dtype=2), dict(y_dtype=1), dict(x=None), dict(y=None), dict(w_packed=None),
                dict(layout=2), dict(x_stride=-1), dict(x_dtype=6, x_scales=None), dict(x_dtype=6, x_scales=4096, batch=2),
                dict(x_dtype=6, x_scales=4096, layout=1)):
        assert _product(L, **bad) == -1, bad
    assert _product(L, layout=1, pixels=1) == -1                 # maps of one pixel are rows
    assert _product(L, w_packed=4104) == -2
    many = dict(pixels=4096, k=512, n=512, x_stride=512)          # quantised into the workspace first: it has to be there
    need = 4096 * 512 // 2 + 4096 * 512 // 32
    assert _product(L, **many) == -3 and _product(L, **many, workspace=4096, workspace_bytes=need - 1) == -3
    assert _product(L, **many, workspace=4104, workspace_bytes=need) == -2
    assert _product(L, x_stride=1 << 24) == -4 and _product(L, layout=1, pixels=1 << 24) == -4 and _product(L, pixels=1 << 40) == -4


def test_oracle_mx_by_hand():
    x = np.zeros((1, 33))
    x[0, :8] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.9]      # largest 7.9: scale 2^0, midpoints go to the even code
    x[0, 32] = -48.0                                              # a block of its own: 2^(5 - 2), 48 = 6 * 8
    codes, scales = OM.quantize(x)
    assert scales.tolist() == [[127, 130]]
    assert codes[0, :8].tolist() == [0, 2, 2, 4, 4, 6, 6, 7] and codes[0, 32] == 15
    assert OM.values(x)[0, :8].tolist() == [0, 1, 1, 2, 2, 4, 4, 6] and OM.values(x)[0, 32] == -48
    assert OM.unpack(np.array([[0x21, 0xf0]], np.uint8)).tolist() == [[1, 2, 0, 15]]
    codes, scales = OM.quantize(np.array([[np.nan] + [1.0] * 31, [0.0] * 32]))
    assert scales.tolist() == [[255], [0]] and np.isnan(OM.dequantize(codes, scales, 32)[0]).all()


def test_oracle_order_by_hand():
    """Row 33, block 5 of k = 200: group 1, row 1 of it, step 2, second block; its scale in the first four steps, third of them."""
    packed, scales = np.zeros((4, 2, 2, 32, 16), np.uint8), np.zeros((1, 2, 2, 32, 4), np.uint8)
    packed[2, 1, 1, 1, 3], scales[0, 1, 1, 1, 2] = 7, 9
    p, s, clean = OM.rows_of(packed, scales, 40, 200)
    assert clean and p.shape == (40, 112) and s.shape == (40, 7)
    assert p[33, 5 * 16 + 3] == 7 and s[33, 5] == 9 and int(p.sum()) == 7 and int(s.sum()) == 9
    packed[3, 1, 1] = 1          # block 7 lies beyond k
    assert not OM.rows_of(packed, scales, 40, 200)[2]


def test_oracle_evidence_by_hand():
    r = OC.evidence([[0.0, 0.0, -np.inf], [-np.inf] * 3, [np.log(3), 0.0, np.nan]], [1, 2, 0], 2)
    assert np.allclose(r["logprob"][0], -np.log(2)) and r["logprob"][1] == -np.inf and np.isnan(r["logprob"][2])
    assert np.allclose(r["entropy"][0], np.log(2)) and r["entropy"][1] == 0 and np.isnan(r["entropy"][2])
    assert r["top_index"].tolist() == [[0, 1], [0, 1], [2, 0]]
    r = OC.evidence([[0.5, 0.0, 1.0]], [0], 3, "none")
    assert np.allclose(r["entropy"], np.log(2)) and np.allclose(r["logprob"], np.log(0.5)) and r["top_index"].tolist() == [[2, 0, 1]]
    r = OC.evidence([[0.0, 1000.0]], [1], 1, "sigmoid")
    assert np.allclose(r["entropy"], np.log(2)) and r["logprob"][0] == 0 and r["top_index"].tolist() == [[1]]


def test_traces_are_refused():
    """What the operators' common check says where a trace is under way (entry points: the GPU tests)."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from object_detectors_amd import hip_ops as ops

    def f(t):
        ops._no_gradient("mx_linear", t, None)
        return t + 1
    x = torch.zeros(3)
    f(x)
    with torch.no_grad():
        with pytest.raises(RuntimeError, match="trace"):
            torch.jit.trace(f, x, check_trace=False)
        with pytest.raises(RuntimeError, match="trace"):
            make_fx(f)(x)
    f(x)


def test_tangents_are_refused():
    import torch.autograd.forward_ad as fw
    from object_detectors_amd import hip_ops as ops
    x = torch.zeros(3)
    with torch.no_grad(), fw.dual_level():
        ops._no_gradient("mx_linear", x, None)
        d = fw.make_dual(x, torch.ones_like(x))
        for call in (lambda: ops._no_gradient("mx_linear", d, None), lambda: ops._no_gradient("mx_linear", x, d)):
            with pytest.raises(RuntimeError, match="no gradient"):
                call()
    ops._no_gradient("mx_linear", x)


def test_alternatives_beyond_the_operators_limit():
    """Refused when the model is built or before anything else is done with a prediction, not halfway; never for models of few classes."""
    from object_detectors_amd.wrapper import Yolov8Core, Yolov8ObbCore, Yolov8PoseCore
    for base in (Yolov8Core, Yolov8PoseCore, Yolov8ObbCore):
        m = base.__new__(base)
        m.device = torch.device("cpu")
        m.model = type("Net", (), {"names": {i: str(i) for i in range(40)}, "kpt_shape": (1, 2)})()
        call = lambda: m.postprocess(torch.zeros(1, 44, 8), torch.zeros(1, 3, 8, 8), [np.zeros((8, 8, 3), np.uint8)], 0.2)
        m.alternatives = 33
        with pytest.raises(ValueError, match="alternatives"):
            call()
        for fine in (32, 0, -1):
            m.alternatives = fine
            with pytest.raises((RuntimeError, ValueError)) as e:
                call()                                    # there is no GPU path here; the count is not what stops it
            assert "alternatives" not in str(e.value)
        m.alternatives = 1000                             # all of them, if they are few
        m.model.names = {0: "a", 1: "b"}
        with pytest.raises((RuntimeError, ValueError)) as e:
            call()
        assert "alternatives" not in str(e.value)


def test_alternatives_beyond_the_limit_at_construction(tmp_path):
    from object_detectors_amd.nets.yolov8 import YoloV8
    from object_detectors_amd.wrapper import Yolov8Core
    names = {i: str(i) for i in range(40)}
    path = str(tmp_path / "w.pt")
    torch.save({"format": "lmi-yolov8-torch", "scale": "n", "nc": 40, "seg": False, "names": names, "state_dict": YoloV8("n", 40, names=names).state_dict()}, path)

    class Model(Yolov8Core):
        alternatives = 33
    with pytest.raises(ValueError, match="alternatives"):
        Model.__new__(Model)._init(path, device="cpu")


def test_activations_that_the_products_lack_stay_as_they_are(monkeypatch):
    """quantize_pointwise replaces what the quantised layer can stand for, and nothing else."""
    from object_detectors_amd.nets.yolov8 import ConvBNAct, MxPointwise, YoloV8
    with pytest.raises(TypeError, match="ReLU"):
        m = ConvBNAct(8, 8).eval()
        m.act = torch.nn.ReLU()
        MxPointwise.of(m)
    net = YoloV8("n", 2).eval()
    mine = [m for name, m in net.named_modules() if isinstance(m, ConvBNAct) and m.conv.kernel_size == (1, 1) and not name.startswith("head")]
    for i, m in enumerate(mine):
        m.act = torch.nn.ReLU() if i % 3 == 0 else torch.nn.Identity() if i % 3 == 1 else m.act
    taken = []
    monkeypatch.setattr(MxPointwise, "of", classmethod(lambda cls, m: taken.append(m) or torch.nn.Identity()))
    assert net.quantize_pointwise() == len(taken) == sum(i % 3 != 0 for i in range(len(mine)))
    assert all(m not in taken and any(m is q for q in net.modules()) for m in mine[::3])


def test_padded_convolutions_stay_as_they_are(monkeypatch):
    from object_detectors_amd.nets.yolov8 import ConvBNAct, MxPointwise, YoloV8
    padded = torch.nn.Conv2d(8, 8, 1, padding=1)
    with pytest.raises(TypeError, match="1x1"):
        MxPointwise.of(padded)
    with pytest.raises(TypeError, match="1x1"):
        MxPointwise.of(torch.nn.Conv2d(8, 8, 3))
    net = YoloV8("n", 2).eval()
    mine = [m for name, m in net.named_modules() if isinstance(m, ConvBNAct) and m.conv.kernel_size == (1, 1) and not name.startswith("head")]
    mine[0].conv.padding = (1, 1)
    mine[1].conv.padding = (0, 2)
    mine[2].conv = torch.nn.Conv2d(mine[2].conv.in_channels, mine[2].conv.out_channels, 1, bias=False, padding="same")     # adds nothing
    taken = []
    monkeypatch.setattr(MxPointwise, "of", classmethod(lambda cls, m: taken.append(m) or torch.nn.Identity()))
    assert net.quantize_pointwise() == len(taken) == len(mine) - 2
    assert mine[0] not in taken and mine[1] not in taken and mine[2] in taken


def test_results_over_inputs_at_the_entry_point(L):
    """Addresses alone decide: nothing is launched."""
    def status(**kw):
        return _probs(L, classes=10, n0=2, n1=4, stride0=40, stride1=10, **kw)
    x, last = 4096, 4096 + 4 * 80                       # fp32 rows of ten, 2 x 4 of them
    free = last + 4096
    for bad in (dict(entropy=x), dict(entropy=last - 4), dict(logprob=x - 4 * 8 + 4), dict(top=1, top_index=x + 8), dict(top=1, top_logprob=x),
                dict(entropy=free, labels=free + 28, label_dtype=4, label_stride0=4, label_stride1=1), dict(entropy=free, count=free + 8),
                dict(entropy=free, index=free - 28, index_range=3), dict(entropy=free, logprob=free + 4), dict(top=2, top_logprob=free, top_index=free + 60),
                dict(entropy=free + 4 * 40, index=free + 4096, index_range=1 << 40), dict(entropy=free, labels=free + 64, label_dtype=5, label_stride0=-5, label_stride1=-1)):
        assert status(**bad) == -1, bad
        assert b"memory of" in L.load().lmi_last_error(), bad
