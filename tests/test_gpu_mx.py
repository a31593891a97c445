"""MXFP4: quantising against the fp64 oracle bit for bit, products within the error bound of an fp32 sum."""
import numpy as np
import pytest
import torch

from oracle import mx as OM

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _ops():
    from object_detectors_amd import hip_ops
    return hip_ops


def _np(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def _same_blocks(q, x):
    """Scales equal everywhere, codes wherever the scale is a number, zeros in what fills up the last group and step."""
    codes, scales = OM.quantize(_np(x).reshape(-1, x.shape[-1]))
    packed, got, clean = OM.rows_of(q.packed.cpu().numpy(), q.scales.cpu().numpy(), codes.shape[0], x.shape[-1])
    assert clean and np.array_equal(got, scales)
    live = np.repeat(scales != 255, 32, axis=1)
    assert np.array_equal(OM.unpack(packed)[live], codes[live])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 31), (2, 32), (5, 33), (64, 80), (7, 400), (130, 2560), (1, 5000), (2049, 96)])
def test_quantize(rows, k, dtype):
    g = torch.Generator().manual_seed(rows * 7 + k)
    x = torch.randn(rows, k, generator=g) * torch.exp2(torch.randint(-8, 9, (rows, 1), generator=g).float())
    x = x.to(DTYPES[dtype]).cuda()
    q = _ops().mx_quantize(x)
    _same_blocks(q, x)
    want = OM.values(_np(x))
    for out in DTYPES.values():       # scale 2^e x {0 .. 6}: exact in every type here (fp16: exponents within its range)
        assert np.array_equal(_np(_ops().mx_dequantize(q, out)), torch.from_numpy(want).to(out).double().numpy())


def test_quantize_every_step():
    """Every midpoint and its neighbours at several scales, subnormals, the ends of the range, zeros, non-finite blocks."""
    u = np.concatenate([np.arange(0, 8, 0.25), np.nextafter(np.arange(0.25, 8, 0.25, dtype=np.float32), np.float32(9)),
                        np.nextafter(np.arange(0.25, 8, 0.25, dtype=np.float32), np.float32(0))]).astype(np.float32)
    rows = []
    for e in (-126, -125, -60, -1, 0, 1, 90, 125):
        v = (u * np.float32(2.0) ** e).astype(np.float32)
        for i in range(0, len(v), 30):
            part = v[i:i + 30]
            rows.append(np.concatenate([part, -part[:32 - len(part)], np.zeros(max(0, 32 - 2 * len(part)), np.float32)])[:32])
    tiny = np.full(32, np.float32(1e-45)); tiny[3] = -7e-45
    odd = [np.zeros(32), -np.zeros(32), tiny, np.full(32, 2.0 ** -127), np.full(32, 3.4028235e38), np.r_[np.inf, np.ones(31)],
           np.r_[np.ones(31), np.nan], np.full(32, -np.inf)]
    x = torch.from_numpy(np.stack(rows + [np.asarray(o, np.float32) for o in odd]).astype(np.float32)).cuda()
    q = _ops().mx_quantize(x)
    _same_blocks(q, x)
    y = _ops().mx_dequantize(q).cpu().numpy()
    want = OM.values(_np(x)).astype(np.float32)
    assert np.array_equal(y, want, equal_nan=True)
    assert np.isnan(y[-3:]).all()


def test_quantize_strides_and_shapes():
    ops = _ops()
    x = torch.randn(6, 10, 100).cuda()
    for v in (x[:, :, 5:77], x[::2], x.transpose(0, 1), x.transpose(1, 2), x[:, 3], x[0, 0], x[:, :, ::2], x[:0]):
        q = ops.mx_quantize(v)
        assert q.shape == v.shape
        if v.numel():
            _same_blocks(q, v)
        assert ops.mx_dequantize(q).shape == v.shape


def _close(got, want, size, k, dtype, act):
    """fp32 sums of k products of at most `size` in all: k + 8 roundings of 2^-24 each at most (2^-23 where the matrix
    instruction cuts instead of rounding); SiLU's slope is below 1.1 and its own error some units; then one rounding to the type."""
    tol = (k + 8) * 2.0 ** -23 * size * (1.1 if act else 1.0)
    if act:
        tol = tol + 8 * 2.0 ** -24 * np.abs(want)
    tol = tol + (np.abs(want) + tol) * torch.finfo(dtype).eps / 2 + (6e-8 if dtype == torch.float16 else 1e-37)
    got = _np(got)
    assert got.shape == want.shape
    both = np.isnan(got) & np.isnan(want)
    assert (np.isnan(got) == np.isnan(want)).all()
    err = np.where(both, 0, np.abs(got - want))
    assert (err <= np.where(both, 0, tol)).all(), (np.nanmax(err), np.nanmax(err / np.maximum(tol, 1e-300)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", [None, "silu"])
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 1280, 1000), (2, 33, 5), (5, 80, 80), (17, 400, 160), (64, 64, 32), (65, 96, 33), (300, 2560, 64),
                                   (1000, 160, 75), (3, 9000, 40), (129, 5000, 130), (700, 640, 640)])
def test_linear(m, k, n, act, dtype):
    ops, dt = _ops(), DTYPES[dtype]
    g = torch.Generator().manual_seed(m + k + n)
    x = (torch.randn(m, k, generator=g) * torch.exp2(torch.randint(-3, 4, (m, 1), generator=g).float())).to(dt).cuda()
    w = torch.randn(n, k, generator=g).cuda() / k ** 0.5
    bias = torch.randn(n, generator=g).cuda() if k % 2 == 0 else None
    wq = ops.mx_quantize(w)
    want, size = OM.product(_np(x), _np(w), None if bias is None else _np(bias), act)
    y = ops.mx_linear(x, wq, bias, act=act)
    assert y.dtype == dt
    _close(y, want, size, k, dt, act)
    z = ops.mx_linear(ops.mx_quantize(x), wq, bias, act=act, dtype=dt)
    _close(z, want, size, k, dt, act)
    out = torch.empty_like(y)
    assert ops.mx_linear(x, wq, bias, act=act, out=out) is out and torch.equal(out, y)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["planes", "channels_last", "slice"])
@pytest.mark.parametrize("b,k,n,h,w,act", [(1, 1, 1, 1, 1, None), (1, 640, 640, 20, 20, "silu"), (3, 400, 75, 7, 13, "silu"), (2, 48, 16, 1, 5, None),
                                           (2, 33, 40, 9, 1, "silu"), (4, 96, 64, 40, 24, None), (1, 80, 32, 160, 96, "silu"), (5, 64, 80, 1, 1, "silu"),
                                           (1, 2600, 70, 3, 11, None), (2, 5000, 33, 4, 4, "silu"),
                                           (2, 48, 40, 160, 128, "silu"), (1, 33, 16, 200, 168, None), (1, 64, 65, 182, 181, "silu"),
                                           (3, 50, 40, 121, 101, "silu"), (2, 200, 330, 83, 61, None), (5, 40, 33, 1, 3, None), (2, 129, 64, 1, 65, "silu")])
def test_pointwise(b, k, n, h, w, act, layout, dtype):
    ops, dt = _ops(), DTYPES[dtype]
    g = torch.Generator().manual_seed(k + n)
    x = torch.randn(b, k, h, w, generator=g).to(dt).cuda()
    if layout == "channels_last":
        x = x.contiguous(memory_format=torch.channels_last)
    elif layout == "slice":           # channels k.. of a map twice as deep, as `chunk` leaves them
        x = torch.cat([torch.full_like(x, float("nan")), x], 1)[:, k:]
    wt = torch.randn(n, k, generator=g).cuda() / k ** 0.5
    bias = torch.randn(n, generator=g).cuda()
    y = ops.mx_pointwise(x, ops.mx_quantize(wt), bias, act=act)
    assert y.shape == (b, n, h, w) and y.dtype == dt
    if layout == "channels_last" and h * w > 1 and k > 1:
        assert y.is_contiguous(memory_format=torch.channels_last)
    want, size = OM.product(_np(x.permute(0, 2, 3, 1)).reshape(-1, k), _np(wt), _np(bias), act)
    _close(y.permute(0, 2, 3, 1).reshape(-1, n), want, size, k, dt, act)


def test_pointwise_odd_strides():
    ops = _ops()
    w = torch.randn(24, 40).cuda()
    wq = ops.mx_quantize(w)
    base = torch.randn(3, 44, 12, 18).half().cuda()
    for x in (base[:, :40, :, 1:], base[:, :40, ::2], base[:, 2:42].transpose(2, 3), base[:, :40, :, :1], base[:, :40, 3:4], base.transpose(0, 1)[:40].transpose(0, 1),
              base[:, :40].flip(3)):
        want, size = OM.product(_np(x.permute(0, 2, 3, 1)).reshape(-1, 40), _np(w))
        _close(ops.mx_pointwise(x, wq).permute(0, 2, 3, 1).reshape(-1, 24), want, size, 40, torch.float16, None)


def test_one_pixel_of_far_images():
    """A pixel of every image of a channels-last batch whose images lie 2^24 elements apart, and of planes."""
    ops = _ops()
    w = torch.randn(20, 256).cuda() / 16
    wq = ops.mx_quantize(w)
    base = torch.randn(3, 256, 1, 1).half().cuda().expand(3, 256, 260, 260)
    for fmt in (torch.channels_last, torch.contiguous_format):
        x = base.contiguous(memory_format=fmt)
        for v in (x[:, :, :1, :1], x[:, :, 259:, 259:]):
            want, size = OM.product(_np(v).reshape(3, 256), _np(w))
            _close(ops.mx_pointwise(v, wq).reshape(3, 20), want, size, 256, torch.float16, None)


def test_non_finite_blocks_stay_in_their_row():
    """A NaN or an infinity makes the results of its own position NaN, and no other's."""
    ops = _ops()
    x = torch.randn(70, 100)
    x[3, 50] = float("nan")
    x[40, 99] = float("inf")
    w = torch.randn(50, 100)
    y = ops.mx_linear(x.cuda(), ops.mx_quantize(w.cuda()))
    bad = torch.isnan(y).cpu()
    assert bad[[3, 40]].all() and bad.sum() == 100
    w[7, 0] = float("-inf")
    bad = torch.isnan(ops.mx_linear(x.cuda(), ops.mx_quantize(w.cuda()))).cpu()
    assert bad[:, 7].all() and bad.sum() == 100 + 68
    p = ops.mx_pointwise(x.t().reshape(1, 100, 70, 1).half().cuda(), ops.mx_quantize(w.cuda()))
    assert torch.isnan(p[0, 7]).all() and int(torch.isnan(p).sum()) == 100 + 68


def test_empty_and_out():
    ops = _ops()
    wq = ops.mx_quantize(torch.randn(8, 32).cuda())
    assert ops.mx_linear(torch.empty(0, 32).cuda(), wq).shape == (0, 8)
    assert ops.mx_linear(ops.mx_quantize(torch.empty(0, 32).cuda()), wq).shape == (0, 8)
    assert ops.mx_pointwise(torch.empty(2, 32, 0, 4).cuda(), wq).shape == (2, 8, 0, 4)
    x = torch.randn(2, 32, 6, 6).cuda()
    guard = torch.full((2 * 8 * 36 + 64,), 5.0).cuda()          # nothing is written beside the result
    out = guard[32:32 + 2 * 8 * 36].view(2, 8, 6, 6)
    ops.mx_pointwise(x, wq, out=out)
    assert (guard[:32] == 5).all() and (guard[-32:] == 5).all()
    assert torch.equal(out, ops.mx_pointwise(x, wq))


def test_captured_and_replayed():
    ops = _ops()
    wq = ops.mx_quantize(torch.randn(64, 96).cuda())
    big = ops.mx_quantize(torch.randn(640, 1280).cuda())
    x, r = torch.randn(2, 96, 10, 10).half().cuda(), torch.randn(1, 1280).half().cuda()

    def step():
        return ops.mx_pointwise(x, wq, act="silu"), ops.mx_linear(r, big), ops.mx_linear(ops.mx_quantize(x.permute(0, 2, 3, 1)), wq)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    for i in range(3):
        x.copy_(torch.randn(2, 96, 10, 10))
        r.copy_(torch.randn(1, 1280))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(res, step()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,n,act", [(2100, 200, 333, "silu"), (1300, 160, 640, None), (130, 1000, 4000, None), (5000, 129, 257, "silu")])
def test_many_rows_and_weights(m, k, n, act, dtype):
    """Rows that are quantised once before the product: the same bits as from an MxTensor, whatever their stride and alignment."""
    ops, dt = _ops(), DTYPES[dtype]
    g = torch.Generator().manual_seed(m + n)
    base = torch.randn(m, k + 11, generator=g).to(dt).cuda()
    w = torch.randn(n, k, generator=g).cuda() / k ** 0.5
    bias = torch.randn(n, generator=g).cuda()
    wq = ops.mx_quantize(w)
    for x in (base[:, 3:3 + k], base[:, :k].contiguous()):
        y = ops.mx_linear(x, wq, bias, act=act)
        want, size = OM.product(_np(x), _np(w), _np(bias), act)
        _close(y, want, size, k, dt, act)
        assert torch.equal(y, ops.mx_linear(ops.mx_quantize(x), wq, bias, act=act, dtype=dt))


@pytest.mark.parametrize("m,n", [(5003, 165), (9001, 700)])
@pytest.mark.parametrize("k", [33, 65, 192, 257, 321, 448, 512])
def test_many_quantised_rows(m, n, k):
    """One to eight steps of 64 along k, rows and weight rows that end inside a tile; either number of rows per workgroup."""
    ops = _ops()
    g = torch.Generator().manual_seed(m + k)
    x, w = torch.randn(m, k, generator=g).cuda(), torch.randn(n, k, generator=g).cuda()
    bias = torch.randn(n, generator=g).cuda()
    guard = torch.full((m * n + 64,), 5.0, dtype=torch.bfloat16, device="cuda")
    y = ops.mx_linear(ops.mx_quantize(x), ops.mx_quantize(w), bias, dtype=torch.bfloat16, out=guard[32:32 + m * n].view(m, n))
    want, size = OM.product(_np(x), _np(w), _np(bias))
    _close(y, want, size, k, torch.bfloat16, None)
    assert (guard[:32] == 5).all() and (guard[-32:] == 5).all()


@pytest.mark.parametrize("step", [1, 2])
def test_many_channels_last_images(step):
    """Images whose rows follow each other, and every other image, whose rows do not."""
    ops = _ops()
    base = torch.randn(6, 192, 24, 26).half().cuda().contiguous(memory_format=torch.channels_last)
    x = base[::step]
    w = torch.randn(400, 192).cuda() / 14
    want, size = OM.product(_np(x.permute(0, 2, 3, 1)).reshape(-1, 192), _np(w), None, "silu")
    y = ops.mx_pointwise(x, ops.mx_quantize(w), act="silu")
    assert y.is_contiguous(memory_format=torch.channels_last)
    _close(y.permute(0, 2, 3, 1).reshape(-1, 400), want, size, 192, torch.float16, "silu")


def _room(gb):
    if torch.cuda.mem_get_info()[0] < gb << 30:
        pytest.skip(f"needs {gb} GB")


def test_far_rows():
    """Inputs, quantised blocks and results beyond 2^32 bytes."""
    _room(48)
    ops = _ops()
    k, m = 1 << 16, (1 << 17) + 40
    x = torch.zeros(m, k, dtype=torch.float16, device="cuda")          # 17 GB, 4.3 GB of blocks
    x[-9:].copy_(torch.randn(9, k))
    want = OM.values(_np(x[-9:]))
    q = ops.mx_quantize(x)
    y = ops.mx_dequantize(q, torch.float16)
    assert np.array_equal(_np(y[-9:]), want) and not y[-100:-9].any()
    ones = ops.mx_quantize(torch.ones(1, k, device="cuda"))            # sums of rows
    for z in (ops.mx_linear(q, ones), ops.mx_linear(x, ones)):
        _close(z[-9:], want.sum(1, keepdims=True), np.abs(want).sum(1, keepdims=True), k, z.dtype, None)
        assert not z[:-9].any()


def test_far_results():
    _room(16)
    ops = _ops()
    x, w = torch.randn(40000, 70).half().cuda(), torch.randn((1 << 16) + 8, 70).cuda()
    y = ops.mx_linear(x, ops.mx_quantize(w))                            # 5.2 GB
    want, size = OM.product(_np(x[-4:]), _np(w[-70:]))
    _close(y[-4:, -70:], want, size, 70, torch.float16, None)


def test_far_maps():
    """Planes and images beyond 2^32 bytes."""
    _room(32)
    ops = _ops()
    x = torch.zeros(9, 640, 700, 702, dtype=torch.float16, device="cuda")   # 5.7 GB
    x[-1].copy_(torch.randn(640, 700, 702))
    w = torch.randn(8, 640).cuda() / 25
    y = ops.mx_pointwise(x, ops.mx_quantize(w))
    part = _np(x[-1, :, -2:]).reshape(640, -1).T
    want, size = OM.product(part, _np(w))
    _close(y[-1, :, -2:].reshape(8, -1).t(), want, size, 640, torch.float16, None)
    assert not y[:-1].any()
    big = torch.randn(1, 70, 2000, 2002).half().cuda()                     # channels 8 MB apart; 5.2 GB of results
    wb = torch.randn(650, 70).cuda()
    z = ops.mx_pointwise(big, ops.mx_quantize(wb))
    want, size = OM.product(_np(big[0, :, -1]).T, _np(wb))
    _close(z[0, :, -1].t(), want, size, 70, torch.float16, None)


def test_odd_maps_end_where_they_end():
    """Planes of odd size, the last ending with its allocation's last element, at addresses that are no multiple of a pair."""
    ops = _ops()
    for k, n, h, w in ((40, 24, 7, 9), (64, 40, 181, 183), (130, 70, 61, 83)):
        wt = torch.randn(n, k).cuda() / k ** 0.5
        wq = ops.mx_quantize(wt)
        for dt in DTYPES.values():
            buf = torch.full((1 + 2 * k * h * w,), float("nan"), dtype=dt, device="cuda")
            x = buf[1:].view(2, k, h, w)
            x.copy_(torch.randn(2, k, h, w))
            guard = torch.full((2 * n * h * w + 3,), 5.0, dtype=dt, device="cuda")
            y = ops.mx_pointwise(x, wq, out=guard[1:-2].view(2, n, h, w))
            want, size = OM.product(_np(x.permute(0, 2, 3, 1)).reshape(-1, k), _np(wt))
            _close(y.permute(0, 2, 3, 1).reshape(-1, n), want, size, k, dt, None)
            assert guard[0] == 5 and (guard[-2:] == 5).all()


def test_graphs_side_by_side():
    """Two captured graphs of products with workspaces, replayed at the same time on two streams."""
    ops = _ops()
    wq = ops.mx_quantize(torch.randn(640, 320).cuda())
    xs = [torch.randn(3000, 320).half().cuda() for _ in range(2)]
    for x in xs:
        ops.mx_linear(x, wq)
    torch.cuda.synchronize()
    graphs, res = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res.append([ops.mx_linear(x, wq, act="silu") for _ in range(4)])
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in xs]
    for i in range(3):
        for x in xs:
            x.copy_(torch.randn(3000, 320))
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for x, r in zip(xs, res):
            want = ops.mx_linear(x, wq, act="silu")
            assert all(torch.equal(t, want) for t in r)


def test_out_over_x_is_refused():
    ops = _ops()
    wq = ops.mx_quantize(torch.randn(64, 64).cuda())
    x, m = torch.randn(10, 64).cuda(), torch.randn(2, 64, 4, 4).cuda()
    cl = m.contiguous(memory_format=torch.channels_last)
    for call in (lambda: ops.mx_linear(x, wq, out=x), lambda: ops.mx_linear(x[:6], wq, out=x[4:]), lambda: ops.mx_pointwise(m, wq, out=m),
                 lambda: ops.mx_pointwise(cl, wq, out=cl)):
        with pytest.raises(ValueError, match="memory of x"):
            call()
    assert torch.equal(ops.mx_linear(x[:5], wq, out=x[5:]), ops.mx_linear(x[:5].clone(), wq))
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.mx_linear(x, wq, torch.zeros(64, device="cuda", requires_grad=True))


def test_refusals():
    ops = _ops()
    x, w = torch.randn(4, 64).cuda(), ops.mx_quantize(torch.randn(8, 64).cuda())
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.mx_linear(x.clone().requires_grad_(), w)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.mx_quantize(x.clone().requires_grad_())
    with torch.no_grad():
        ops.mx_linear(x.clone().requires_grad_(), w)
    for err, call in ((TypeError, lambda: ops.mx_quantize(x.int())), (TypeError, lambda: ops.mx_linear(x.double(), w)),
                      (TypeError, lambda: ops.mx_linear(x, torch.randn(8, 64).cuda())), (ValueError, lambda: ops.mx_linear(x[:, :63], w)),
                      (ValueError, lambda: ops.mx_linear(x, w, act="relu")), (ValueError, lambda: ops.mx_linear(x, w, dtype=torch.float16)),
                      (ValueError, lambda: ops.mx_linear(x, w, torch.zeros(7).cuda())), (ValueError, lambda: ops.mx_linear(x, w, torch.zeros(8).cuda().half())),
                      (ValueError, lambda: ops.mx_linear(x, w, torch.zeros(8))), (ValueError, lambda: ops.mx_linear(x, w, out=torch.empty(4, 9).cuda())),
                      (ValueError, lambda: ops.mx_pointwise(x, w)), (ValueError, lambda: ops.mx_pointwise(torch.randn(1, 32, 4, 4).cuda(), w)),
                      (ValueError, lambda: ops.mx_linear(x, w, out=torch.empty(8, 4).cuda().t())), (ValueError, lambda: ops.mx_quantize(x[:, :0])),
                      (TypeError, lambda: ops.mx_dequantize(x)), (TypeError, lambda: ops.mx_dequantize(w, torch.int8))):
        with pytest.raises(err):
            call()


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_of_single_images_and_channels(dtype):
    """Strides of dimensions of one element say nothing, however large: a pixel of one far-strided image, one channel of planes and of
    channels-last maps, single images of every layout."""
    ops = _ops()
    g = torch.Generator().manual_seed(3)
    dt = DTYPES[dtype]
    big = torch.zeros(1, 160, 160, 1280, dtype=dt, device="cuda")
    big[:, 5, 7] = torch.randn(1280, generator=g).to(dt).cuda()
    pixel = big.permute(0, 3, 1, 2)[:, :, 5:6, 7:8]
    assert pixel.stride()[0] >= 1 << 24 and pixel.is_contiguous()
    few = torch.randn(2, 3, 5, 7, generator=g).to(dt).cuda()
    wide = lambda h, w: torch.as_strided(few, (1, 1, h, w), (1 << 25, 1 << 26, w, 1))
    views = [pixel, wide(5, 7), wide(1, 6), wide(6, 1), wide(1, 1), torch.as_strided(few, (2, 1, 3, 5), (105, 1 << 27, 7, 1)),
             torch.as_strided(few, (2, 1, 1, 1), (105, 1 << 27, 1 << 26, 1 << 25)), torch.as_strided(few, (1, 3, 5, 7), (1 << 30, 1, 21, 3)),
             few[:1], few[:1].contiguous(memory_format=torch.channels_last)]
    for v in views:
        b, k, h, w = v.shape
        weight = torch.randn(21, k, generator=g).cuda() / k ** 0.5
        want, size = OM.product(_np(v.permute(0, 2, 3, 1)).reshape(-1, k), _np(weight))
        got = ops.mx_pointwise(v, ops.mx_quantize(weight))
        assert got.shape == (b, 21, h, w)
        _close(got.permute(0, 2, 3, 1).reshape(-1, 21), want, size, k, dt, None)


def test_results_over_weights_and_biases_are_refused():
    ops = _ops()
    w = torch.randn(64, 64).cuda()
    wq, bias = ops.mx_quantize(w), torch.randn(64).cuda()
    x, m = torch.randn(1, 64).cuda(), torch.randn(1, 64, 4, 4).cuda()
    over = wq.packed.view(-1).view(torch.float32)
    scales = wq.scales.view(-1).view(torch.float32)
    for call in (lambda: ops.mx_linear(x, wq, bias, out=bias.view(1, 64)), lambda: ops.mx_linear(x, wq, out=over[:64].view(1, 64)),
                 lambda: ops.mx_linear(x, wq, out=scales[64:].view(1, 64)), lambda: ops.mx_pointwise(m[:, :, :1, :1], wq, bias, out=bias.view(1, 64, 1, 1)),
                 lambda: ops.mx_pointwise(m[:, :, :1, 1:2], wq, out=over[:64].view(1, 64, 1, 1))):
        with pytest.raises(ValueError, match="memory of"):
            call()


def test_tracing_is_refused():
    """A trace would hold the allocation of the result and not the product."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from object_detectors_amd.nets.yolov8 import ConvBNAct, MxPointwise
    ops = _ops()
    x = torch.randn(1, 64, 4, 4).cuda()
    net = torch.nn.Sequential(MxPointwise.of(ConvBNAct(64, 32).eval().cuda())).eval()
    with torch.no_grad():
        want = net(x)
        with pytest.raises(RuntimeError, match="trace"):
            torch.jit.trace(net, x, check_trace=False)
        assert torch.equal(net(x), want)                  # and nothing stays behind
    q = ops.mx_quantize(torch.randn(8, 64).cuda())
    for f in (lambda t: ops.class_logprobs(t)["entropy"], lambda t: ops.mx_dequantize(ops.mx_quantize(t)), lambda t: ops.mx_linear(t, q)):
        with pytest.raises(RuntimeError, match="trace"):
            torch.jit.trace(f, torch.randn(3, 64).cuda(), check_trace=False)
        with pytest.raises(RuntimeError, match="trace"):
            make_fx(f)(torch.randn(3, 64).cuda())


def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fw
    ops = _ops()
    x, w = torch.randn(4, 64).cuda(), ops.mx_quantize(torch.randn(8, 64).cuda())
    with torch.no_grad(), fw.dual_level():
        d = fw.make_dual(x, torch.ones_like(x))
        bias = fw.make_dual(torch.zeros(8).cuda(), torch.ones(8).cuda())
        maps = d.view(1, 64, 2, 2)
        for call in (lambda: ops.class_logprobs(d), lambda: ops.mx_quantize(d), lambda: ops.mx_linear(d, w), lambda: ops.mx_linear(x, w, bias),
                     lambda: ops.mx_pointwise(maps, w)):
            with pytest.raises(RuntimeError, match="no gradient"):
                call()
        ops.mx_linear(x, w)                               # what carries no tangent passes
