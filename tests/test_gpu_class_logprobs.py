"""class_logprobs against the fp64 oracle: types, layouts, lengths, masked rows, ties, gathered rows."""
import numpy as np
import pytest
import torch

from oracle import class_logprobs as OC

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ULP = 2.0 ** -24


def _ops():
    from object_detectors_amd import hip_ops
    return hip_ops


def _check(res, x, labels, top, activation, sequential=160):
    """Tolerances, from the arithmetic: every sum runs over at most `sequential` terms one after another (a lane's share plus the
    tree over the lanes), each of them with a relative error of a few units (2^-24); the exponential's argument is rounded
    once (relative error 2 |z| units of e^z, and sum p|z| <= ln C over a row)."""
    x = x.detach().float().cpu().numpy()
    ref = OC.evidence(x, None if labels is None else labels.cpu().numpy(), top, activation)
    c = x.shape[-1]
    lnc = np.log(c) + 1
    with np.errstate(all="ignore"):
        if activation == "softmax":
            unit = (sequential + 8 + 4 * lnc) * ULP
            tol_h = unit * (2 + 2 * lnc)
            tol_lp = lambda v: unit + 4 * ULP * np.abs(v)
        else:
            # an answer's entropy has a relative error of some units, |x| more of them through e^-|x| (fp64 of x: the score's logit)
            a = np.abs(x.astype(np.float64)) if activation == "sigmoid" else np.zeros_like(x, np.float64)
            h = OC.evidence(x[..., None], None, 0, activation)["entropy"]
            tol_h = np.where(np.isfinite(a), h * (2 * a + 12 + sequential) * ULP, 0).sum(-1)
            tol_lp = lambda v: 8 * ULP * np.abs(v) + 2.0 ** -140
    got = {k: v.cpu().numpy() for k, v in res.items()}
    assert set(got) == set(ref)

    def close(a, b, tol):
        same = (a == b) | (np.isnan(a) & np.isnan(b))
        with np.errstate(all="ignore"):
            err = np.where(same, 0, np.abs(a.astype(np.float64) - b))
        assert not np.isnan(err).any() and (err <= np.where(same, 0, tol)).all(), np.nanmax(err - tol)

    close(got["entropy"], ref["entropy"], tol_h)
    if labels is not None:
        close(got["logprob"], ref["logprob"], tol_lp(ref["logprob"]))
    if top:
        assert np.array_equal(got["top_index"], ref["top_index"])
        close(got["top_logprob"], ref["top_logprob"], tol_lp(ref["top_logprob"]))


def _rows(seed, n, c, dtype, activation, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, c, generator=g) * scale
    if activation == "none":
        x = torch.sigmoid(x)
    return x.to(dtype).cuda(), torch.randint(0, c, (n,), generator=g).cuda()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("activation", ["softmax", "sigmoid", "none"])
@pytest.mark.parametrize("n,c,top", [(1, 1, 1), (3, 2, 2), (7, 8, 0), (5, 9, 9), (300, 80, 5), (2, 1000, 32), (4, 1021, 7), (3, 1025, 3),
                                     (5, 4099, 16), (3, 8192, 0), (130, 8193, 1), (129, 16500, 10), (2, 40003, 32), (1, 270001, 20)])
def test_rows(n, c, top, activation, dtype):
    x, labels = _rows(n * 1000 + c, n, c, DTYPES[dtype], activation)
    _check(_ops().class_logprobs(x, labels, top=top, activation=activation), x, labels, top, activation)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("activation", ["softmax", "sigmoid", "none"])
@pytest.mark.parametrize("b,g,c,a,top", [(1, 1, 1, 1, 1), (2, 4, 16, 525, 2), (3, 1, 80, 1701, 5), (1, 2, 63, 4097, 32), (2, 1, 300, 2100, 8),
                                         (1, 1, 200, 70, 4)])
def test_planes(b, g, c, a, top, activation, dtype):
    """Class planes (the head's layout, distance bins): classes lie `a` apart."""
    gen = torch.Generator().manual_seed(c)
    planes = torch.randn(b, g * c, a, generator=gen) * 2
    if activation == "none":
        planes = torch.sigmoid(planes)
    x = planes.to(DTYPES[dtype]).cuda().view(b, g, c, a).transpose(2, 3)
    labels = torch.randint(0, c, (b, g, a), generator=gen).to(torch.int32).cuda()
    _check(_ops().class_logprobs(x, labels, top=min(top, c), activation=activation), x, labels, min(top, c), activation, sequential=c + 8)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,g,c,a,top,activation", [(2, 1, 63, 8201, 32, "softmax"), (4, 1, 39, 8201, 8, "softmax"), (1, 4, 16, 4200, 2, "softmax"), (1, 1, 80, 16400, 2, "none"),
                                                    (3, 1, 33, 5500, 0, "sigmoid"), (16, 1, 70, 8200, 5, "softmax"), (4, 1, 300, 4100, 1, "softmax")])
def test_many_planes(b, g, c, a, top, activation, dtype):
    test_planes(b, g, c, a, top, activation, dtype)


@pytest.mark.parametrize("c,rows,top", [(5, 24, 3), (20, 16800, 2), (20, 33600, 7), (64, 16800, 20), (70, 132000, 5)])
def test_many_planes_of_odd_values(c, rows, top):
    """The odd values again, in rows that lie side by side, so many that each has a thread of its own."""
    x, gen = _odd_rows(c)
    labels = torch.randint(0, c, (12,), generator=gen)
    planes = x.t().repeat(1, rows // 12).contiguous().cuda()
    r = _ops().class_logprobs(planes.t(), labels.repeat(rows // 12).cuda(), top=top)
    _check({k: v[:12] for k, v in r.items()}, x, labels, top, "softmax", sequential=c + 8)
    for v in r.values():
        v = v.reshape(rows // 12, -1).nan_to_num(nan=123.0)
        assert (v == v[0]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,nc,a,m,top,activation", [(1, 80, 8400, 300, 5, "none"), (4, 3, 525, 17, 3, "sigmoid"), (2, 131, 1701, 64, 32, "softmax"),
                                                     (2, 1, 40, 5, 1, "none")])
def test_gathered(b, nc, a, m, top, activation, dtype):
    """Rows at NMS anchors, labels from the class column of the NMS rows, per-image counts; rows behind a count stay."""
    gen = torch.Generator().manual_seed(nc)
    head = torch.randn(b, 4 + nc + 3, a, generator=gen) * 2
    if activation == "none":
        head = torch.sigmoid(head)
    head = head.to(DTYPES[dtype]).cuda()
    index = torch.randint(0, a, (b, m), generator=gen).to(torch.int32).cuda()
    index[:, -1] = index[:, 0]     # the same anchor twice
    count = torch.tensor([m, 0, m // 2, 1][:b], dtype=torch.int32).cuda()
    det = torch.randn(b, m, 9, generator=gen).cuda()
    det[:, :, 5] = torch.randint(0, nc, (b, m), generator=gen).float().cuda()
    out = {"logprob": torch.full((b, m), 7.0).cuda(), "entropy": torch.full((b, m), 7.0).cuda(),
           "top_logprob": torch.full((b, m, top), 7.0).cuda(), "top_index": torch.full((b, m, top), 7, dtype=torch.int32).cuda()}
    res = _ops().class_logprobs(head[:, 4:4 + nc].transpose(1, 2), det[:, :, 5], top=top, activation=activation, index=index, count=count, out=out)
    assert all(res[k] is out[k] for k in out)
    for i in range(b):
        n = int(count[i])
        x = head[i, 4:4 + nc].t()[index[i, :n].long()]
        if n:
            _check({k: v[i, :n] for k, v in res.items()}, x, det[i, :n, 5].long(), top, activation)
        for v in res.values():
            assert (v[i, n:] == 7).all()


def _odd_rows(c):
    gen = torch.Generator().manual_seed(c)
    x = torch.randn(12, c, generator=gen)
    x[1, torch.rand(c, generator=gen) < 0.9] = -float("inf")
    x[2] = -float("inf")                                  # nothing left
    x[3] = torch.finfo(torch.float32).min                 # masked by the lowest value, all of it
    x[4, 1:] = torch.finfo(torch.float32).min
    x[5] = 1.5                                            # all equal
    x[6] = torch.randint(0, 3, (c,), generator=gen).float()
    x[7, c // 2] = float("nan")
    x[8, c // 2] = float("inf")
    x[9] = torch.tensor([0.0, -0.0]).repeat((c + 1) // 2)[:c]
    x[10] = -float("inf")
    x[10, c - 1] = 3.0                                    # one class left
    x[11] = torch.arange(c).flip(0) * 0.001               # sorted
    return x, gen


@pytest.mark.parametrize("c", [5, 100, 1500, 20000, 70000])
@pytest.mark.parametrize("layout", ["rows", "planes"])
def test_masked_and_odd_values(c, layout):
    """Masked classes, rows with nothing left, the type's lowest value as a mask, equal values, infinities and NaN."""
    x, gen = _odd_rows(c)
    x = x.cuda()
    if layout == "planes":
        x = x.t().contiguous().t()
    labels = torch.randint(0, c, (12,), generator=gen).cuda()
    for top in (0, min(c, 4), min(c, 32)):
        _check(_ops().class_logprobs(x, labels, top=top), x, labels, top, "softmax", sequential=160 if layout == "rows" or c > 64 else c + 8)
    _check(_ops().class_logprobs(x, labels, top=2, activation="sigmoid"), x, labels, 2, "sigmoid")


def test_probabilities_at_the_borders():
    x = torch.tensor([[0.0, 1.0, 0.5, 2.0 ** -24, 1 - 2.0 ** -24, 6e-8], [0.0] * 6, [1.0] * 6, [0.5, float("nan"), 0.25, 0.1, 0.2, 0.3]]).cuda()
    for label in range(6):
        labels = torch.full((4,), label).cuda()
        _check(_ops().class_logprobs(x, labels, top=6, activation="none"), x, labels, 6, "none")


def test_many_best_in_few_lanes():
    """The best values sit where a few lanes hold them all (every 64th group of a tile): the candidate table overflows."""
    for n, c in ((1, 8000), (2, 16000), (3, 900)):
        x = torch.randn(n, c)
        at = torch.arange(c)
        x[:, (at // 8) % 64 == 5] += 100.0
        x = x.bfloat16().cuda()
        labels = torch.zeros(n, dtype=torch.int64).cuda()
        _check(_ops().class_logprobs(x, labels, top=32), x, labels, 32, "softmax")


def test_labels_and_shapes():
    ops = _ops()
    x, labels = _rows(1, 6, 50, torch.float32, "softmax")
    bad = torch.tensor([-1, 50, 3, 1 << 40, -(1 << 40), 0]).cuda()
    _check(ops.class_logprobs(x, bad), x, bad, 0, "softmax")
    lp = ops.class_logprobs(x, torch.tensor([float("nan"), 1.0, -3.0, 1e20, 49.0, 50.0]).cuda())["logprob"].cpu()
    assert torch.isnan(lp[[0, 2, 3, 5]]).all() and not torch.isnan(lp[[1, 4]]).any()
    assert set(ops.class_logprobs(x)) == {"entropy"}
    one = ops.class_logprobs(x[0], labels[0], top=3)                      # a single row without leading dimensions
    assert one["entropy"].shape == () and one["top_index"].shape == (3,)
    empty = ops.class_logprobs(x[:0], labels[:0], top=3)
    assert empty["entropy"].shape == (0,) and empty["top_index"].shape == (0, 3)
    wide = torch.randn(4, 3, 5, 64).cuda().permute(2, 0, 1, 3)            # strides two of which cannot say: copied
    lab = torch.randint(0, 64, (5, 4, 3)).cuda()
    _check(ops.class_logprobs(wide, lab, top=2), wide, lab, 2, "softmax")
    same = x[:1].expand(6, 50)                                            # broadcast rows, broadcast classes
    _check(ops.class_logprobs(same, labels, top=2), same, labels, 2, "softmax")
    flat = x[:, :1].expand(6, 50)
    _check(ops.class_logprobs(flat, labels, top=2), flat, labels, 2, "softmax")
    every = x[:, ::3]                                                     # a class stride that is neither 1 nor a plane
    _check(ops.class_logprobs(every, labels % 17, top=2), every, labels % 17, 2, "softmax")


def test_offset_rows_keep_alignment_rules():
    """Rows that start at every offset inside 16 bytes."""
    base = torch.randn(40000).half().cuda()
    for off in range(9):
        for c in (1, 7, 513, 2049, 9001):
            x = base[off:off + 3 * c].view(3, c)
            labels = torch.tensor([0, c - 1, c // 2]).cuda()
            _check(_ops().class_logprobs(x, labels, top=min(c, 4)), x, labels, min(c, 4), "softmax")


def test_bad_index_gives_nan():
    ops = _ops()
    x = torch.randn(1, 30, 6).cuda()
    index = torch.tensor([[-1, 30, 29, 2 ** 31 - 1, 0]], dtype=torch.int32).cuda()
    r = ops.class_logprobs(x, torch.zeros(1, 5, dtype=torch.int64).cuda(), top=2, index=index)
    for k in ("logprob", "entropy"):
        assert torch.isnan(r[k][0, [0, 1, 3]]).all() and not torch.isnan(r[k][0, [2, 4]]).any()
    assert (r["top_index"][0, [0, 1, 3]] == -1).all() and (r["top_index"][0, [2, 4]] >= 0).all()


def test_far_rows_of_a_large_tensor():
    """Offsets beyond 2^32 bytes and 2^31 elements."""
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("needs 16 GB")
    c, n = 1 << 16, (1 << 15) + 40
    x = torch.zeros(n, c, dtype=torch.float16, device="cuda")
    x[-3:].copy_(torch.randn(3, c))
    labels = torch.arange(3).cuda()
    _check(_ops().class_logprobs(x[-3:], labels, top=3), x[-3:], labels, 3, "softmax")
    r = _ops().class_logprobs(x, torch.zeros(n, dtype=torch.int64, device="cuda"))
    _check({k: v[-3:] for k, v in r.items()}, x[-3:], torch.zeros(3, dtype=torch.int64), 0, "softmax")


def test_more_rows_than_a_grid_holds():
    """2^28 rows of 9 classes, 16 lanes each."""
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("needs 16 GB")
    n = (1 << 28) + 40
    x = torch.zeros(n, 9, dtype=torch.float16, device="cuda")
    x[-5:].copy_(torch.randn(5, 9))
    x[1 << 20].copy_(torch.randn(9))
    r = _ops().class_logprobs(x)["entropy"]
    for at in (slice(n - 9, n), slice((1 << 20) - 2, (1 << 20) + 2)):
        _check({"entropy": r[at]}, x[at], None, 0, "softmax")
    assert int((r == r[0]).sum()) == n - 6


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,c,top", [(2100, 5000, 5), (2050, 17000, 8), (300, 40000, 3), (255, 70003, 6)])
def test_many_long_rows(n, c, top, dtype):
    """Rows that a team goes over in tiles, or in parts, many of them; the last ones are checked."""
    x, labels = _rows(c, n, c, DTYPES[dtype], "softmax")
    r = _ops().class_logprobs(x, labels, top=top)
    _check({k: v[-20:] for k, v in r.items()}, x[-20:], labels[-20:], top, "softmax")


def test_captured_and_replayed():
    ops = _ops()
    x, labels = _rows(3, 2, 50001, torch.float32, "softmax")
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        ops.class_logprobs(x, labels, top=5)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = ops.class_logprobs(x, labels, top=5)
    for i in range(3):
        x.copy_(torch.randn(2, 50001) * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        _check(res, x, labels, 5, "softmax")
        eager = ops.class_logprobs(x, labels, top=5)
        assert all(torch.equal(res[k], eager[k]) for k in res)


def test_two_streams_agree():
    """A long row on two streams at once: the parts' workspaces are the calls' own; the results have the same bits every time."""
    ops = _ops()
    data = [_rows(s, 3, 100003, torch.bfloat16, "softmax") for s in (1, 2)]
    want = [ops.class_logprobs(x, l, top=8) for x, l in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in data]
    got = [[], []]
    for _ in range(10):
        for i, (x, l) in enumerate(data):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.class_logprobs(x, l, top=8))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(r[k], want[i][k]) for k in r)


def test_graphs_side_by_side():
    """Two captured graphs of long rows, whose parts are joined through workspaces, replayed at the same time on two streams."""
    ops = _ops()
    data = [_rows(s, 2, 70001, torch.float16, "softmax") for s in (1, 2)]
    graphs, res = [], []
    for x, l in data:
        ops.class_logprobs(x, l, top=4)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res.append([ops.class_logprobs(x, l, top=4) for _ in range(4)])
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in data]
    for i in range(3):
        for x, _ in data:
            x.copy_(torch.randn(2, 70001) * (i + 1))
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for (x, l), several in zip(data, res):
            want = ops.class_logprobs(x, l, top=4)
            for r in several:
                assert all(torch.equal(r[k], want[k]) for k in r)


def test_count_beyond_the_rows_and_far_labels():
    """count above M means all rows, below zero none; labels of 64 bits that a 32-bit reading would take for classes are none."""
    ops = _ops()
    x = torch.randn(4, 5, 9).cuda()
    labels = torch.tensor([0, 2 ** 32, -2 ** 32 + 3, 8, 9], dtype=torch.int64).repeat(4, 1).cuda()
    count = torch.tensor([99, 0, -3, 2], dtype=torch.int32).cuda()
    full = ops.class_logprobs(x, labels, top=2)
    assert torch.isnan(full["logprob"])[0].tolist() == [False, True, True, False, True]
    out = {k: torch.full_like(v, 77) for k, v in full.items()}
    ops.class_logprobs(x, labels, top=2, count=count, out=out)
    for k, v in full.items():
        for b, rows in enumerate((5, 0, 0, 2)):
            assert torch.equal(out[k][b, :rows].nan_to_num(5), v[b, :rows].nan_to_num(5)) and (out[k][b, rows:] == 77).all()
    planes = x.transpose(1, 2).contiguous().transpose(1, 2)               # the same rows, classes as planes
    out = {k: torch.full_like(v, 77) for k, v in full.items()}
    ops.class_logprobs(planes, labels, top=2, count=count, out=out)
    for b, rows in enumerate((5, 0, 0, 2)):
        assert torch.equal(out["top_index"][b, :rows], full["top_index"][b, :rows]) and all((t[b, rows:] == 77).all() for t in out.values())


def test_refusals():
    ops = _ops()
    x = torch.randn(4, 6, 9).cuda()
    lab = torch.zeros(4, 6, dtype=torch.int64).cuda()
    idx, cnt = torch.zeros(4, 3, dtype=torch.int32).cuda(), torch.zeros(4, dtype=torch.int32).cuda()
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.class_logprobs(x.clone().requires_grad_(), lab)
    for err, call in ((TypeError, lambda: ops.class_logprobs(x.int(), lab)), (ValueError, lambda: ops.class_logprobs(x, lab, top=10)),
                      (ValueError, lambda: ops.class_logprobs(x, lab, top=-1)), (ValueError, lambda: ops.class_logprobs(x, lab, activation="relu")),
                      (ValueError, lambda: ops.class_logprobs(x, lab[:3])), (TypeError, lambda: ops.class_logprobs(x, lab.short())),
                      (TypeError, lambda: ops.class_logprobs(x, lab.cpu())), (ValueError, lambda: ops.class_logprobs(x[..., :0])),
                      (ValueError, lambda: ops.class_logprobs(torch.randn(2, 40).cuda(), top=33)),
                      (ValueError, lambda: ops.class_logprobs(x, index=idx.long())), (ValueError, lambda: ops.class_logprobs(x, index=idx[:3])),
                      (ValueError, lambda: ops.class_logprobs(x[0], index=idx)), (ValueError, lambda: ops.class_logprobs(x, index=idx.t())),
                      (ValueError, lambda: ops.class_logprobs(x, count=cnt[:3])), (ValueError, lambda: ops.class_logprobs(x, count=cnt.long())),
                      (ValueError, lambda: ops.class_logprobs(x, out={})), (ValueError, lambda: ops.class_logprobs(x[0], count=cnt)),
                      (ValueError, lambda: ops.class_logprobs(x, out={"entropy": torch.empty(6, 4).cuda().t()}))):
        with pytest.raises(err):
            call()


def _flat_rows(c):
    """12 rows of c classes where many values are equal or climb slowly -- a long fp32 sum of such terms rounds every one of them the
    same way --, beside a few that differ."""
    gen = torch.Generator().manual_seed(c)
    x = torch.empty(12, c)
    for r, level in enumerate((-0.7, -3.3, -6.1, -8.0, -9.7)):
        x[r] = level
        x[r, (r * 37 + 5) % c] = 0.0                      # one peak above a flat background
    x[5] = 1.3                                            # all equal
    x[6] = torch.linspace(-1, 1, c)                       # climbs
    x[7] = torch.linspace(-12, 9, c)
    x[8] = torch.linspace(9, -12, c)                      # falls
    x[9] = torch.randn(c, generator=gen)
    x[10] = torch.where(torch.rand(c, generator=gen) < 0.9, -float("inf"), 0.7)
    x[11] = torch.linspace(-40, 40, c)
    return x


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("activation", ["softmax", "sigmoid", "none"])
@pytest.mark.parametrize("c,rows,top", [(8009, 16800, 2), (30011, 16800, 1), (4001, 132000, 5)])
def test_long_planes_of_flat_values(c, rows, top, activation, dtype):
    """Thousands of classes as planes, a thread per row: the error does not grow with the number of classes.  `sequential`: 16 terms added one
    after another, the sum of such groups with what each addition loses carried along (4), steps of the maximum below 0.25 likewise, larger
    ones 4 each, the earlier of them fading with e^-0.25 (4 / (1 - e^-0.25) = 18): 64 covers it."""
    x = _flat_rows(c)
    if activation == "none":
        x = torch.sigmoid(x)
    x = x.to(DTYPES[dtype])
    labels = torch.tensor([(r * 37 + 5) % c for r in range(12)])
    planes = x.t().contiguous().cuda().repeat(1, rows // 12)
    r = _ops().class_logprobs(planes.t(), labels.repeat(rows // 12).cuda(), top=top, activation=activation)
    for v in r.values():
        v = v.reshape(rows // 12, -1).nan_to_num(nan=123.0)
        assert (v == v[0]).all()
    _check({k: v[:12] for k, v in r.items()}, x, labels, top, activation, sequential=64)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,c", [(1, (1 << 27) + 1), (3, (1 << 25) + 77), (2049, 400009)])
def test_very_long_flat_rows(rows, c, dtype):
    """The same for rows whose classes lie side by side, by closed forms: a peak of 0 above c - 1 values v; 64 values of a thread's
    added one after another at most, the rest as above.  Entropies of independent classes: c - 1 equal ones and the peak's."""
    dt = DTYPES[dtype]
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("needs 16 GB")
    for level in (-0.703125, -3.3125):                   # exact in all three types
        x = torch.full((1, c), level, dtype=dt, device="cuda")
        x[0, 5] = 0.0
        x = x.expand(rows, c)
        labels = torch.full((rows,), 5, dtype=torch.int64, device="cuda")
        r = _ops().class_logprobs(x, labels)
        s = 1 + (c - 1) * np.exp(level)
        log_s = np.log(s)
        h = log_s - (c - 1) * np.exp(level) * level / s
        unit = (64 + 64 + 8 + 4 * (np.log(c) + 1)) * ULP
        assert (r["logprob"].cpu().double() + log_s).abs().max() <= unit + 4 * ULP * log_s
        assert (r["entropy"].cpu().double() - h).abs().max() <= unit * (2 + 2 * (np.log(c) + 1))
        e = np.log1p(np.exp(level)) - level * np.exp(level) / (1 + np.exp(level))
        r = _ops().class_logprobs(x, labels, activation="sigmoid")
        want = (c - 1) * e + np.log(2)
        assert (r["entropy"].cpu().double() - want).abs().max() <= want * (2 * abs(level) + 12 + 64 + 64) * ULP


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,c,top", [(3, 129, 32), (5, 300, 7), (2, 2100, 32), (2, 20000, 32), (1, 70001, 32), (40, 131, 1)])
def test_values_that_are_no_probabilities(n, c, top, dtype):
    """Values below zero have no logarithm, but an order and a class: the alternatives name classes that exist."""
    x = -1 - torch.rand(n, c, generator=torch.Generator().manual_seed(c))
    x[-1] = 0.0                                           # and a row of zeros
    x[-1, 7] = -0.5
    x = x.to(DTYPES[dtype]).cuda()
    labels = torch.zeros(n, dtype=torch.int64).cuda()
    _check(_ops().class_logprobs(x, labels, top=top, activation="none"), x, labels, top, "none")


def test_results_over_inputs_are_refused():
    ops = _ops()
    x = torch.randn(4, 6, 9).cuda()
    labels, index, count = torch.zeros(4, 6).cuda(), torch.zeros(4, 6, dtype=torch.int32).cuda(), torch.full((4,), 6, dtype=torch.int32).cuda()
    fresh = lambda: {"entropy": torch.zeros(4, 6).cuda(), "logprob": torch.zeros(4, 6).cuda(), "top_logprob": torch.zeros(4, 6, 1).cuda(),
                     "top_index": torch.zeros(4, 6, 1, dtype=torch.int32).cuda()}
    call = lambda out: ops.class_logprobs(x, labels, top=1, index=index, count=count, out=out)
    call(fresh())
    flat = x.view(-1)
    for key, t in (("entropy", flat[20:44].view(4, 6)), ("top_logprob", flat[:24].view(4, 6, 1)), ("logprob", labels), ("top_index", index.unsqueeze(-1)),
                   ("top_index", count.new_zeros(30)[:24].view(4, 6, 1))):
        out = fresh()
        out[key] = t
        if key == "top_index" and t.data_ptr() != index.data_ptr():
            call(out)                                     # a part of a larger tensor is fine
            continue
        with pytest.raises(ValueError, match="memory of"):
            call(out)
    out = fresh()
    out["logprob"] = out["entropy"]                       # two results in one place
    with pytest.raises(ValueError, match="memory of"):
        call(out)
    both = torch.zeros(2, 4, 6).cuda()                    # side by side is fine
    out = dict(fresh(), entropy=both[0], logprob=both[1])
    want = call(fresh())
    assert all(torch.equal(v, want[k]) for k, v in call(out).items())
    one = torch.zeros(1, dtype=torch.int32).cuda()
    with pytest.raises(ValueError, match="memory of"):
        ops.class_logprobs(x[:1, :1], top=1, count=one, out={"entropy": torch.zeros(1, 1).cuda(), "top_logprob": torch.zeros(1, 1, 1).cuda(),
                                                            "top_index": one.view(1, 1, 1)})


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["rows", "planes"])
@pytest.mark.parametrize("c,top", [(100, 3), (131, 1), (600, 5), (5000, 32), (20001, 8), (70001, 32)])
def test_nan_of_the_first_class_among_many_equal_values(c, top, layout, dtype):
    """More candidates than the table holds, the best of them a NaN at class 0."""
    x = torch.full((4, c), -float("inf"))
    x[0, 0] = float("nan")
    x[1] = 0.5
    x[1, [0, c - 1]] = float("nan")
    x[2] = float("nan")
    x[3, 0] = float("inf")
    x = x.to(DTYPES[dtype]).cuda()
    if layout == "planes":
        x = x.t().contiguous().t()
    labels = torch.tensor([0, 1, 2, 0]).cuda()
    _check(_ops().class_logprobs(x, labels, top=top), x, labels, top, "softmax")
