"""The language-model style operators of this package, measured: log probabilities of given classes with their entropy
and the best alternatives, and the MXFP4 format (4-bit elements, one power-of-two scale per block of 32): quantising,
and the products of quantised weights with activations in rows or in planes (1x1 convolutions).

With `own` false every pass is computed by elementary torch operations in fp32; with `own` true by the package's calls."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
BLOCK = 32


# --------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # evidence of one image's detections: head of a seg model at 640 (8400 anchors, 80 classes, 32 coefficients), fp16
        {"name": "evidence_image", "op": "detections", "batch": 1, "nc": 80, "nm": 32, "anchors": 8400, "rows": 300, "top": 5,
         "activation": "none", "dtype": "f16"},
        # the same for the benchmark's batch of 64, fp32 head
        {"name": "evidence_batch", "op": "detections", "batch": 64, "nc": 80, "nm": 32, "anchors": 8400, "rows": 300, "top": 5,
         "activation": "none", "dtype": "f32"},
        # distribution over the 16 distance bins of every box side of a batch of 64: how sure the box edges are
        {"name": "bins_batch", "op": "planes", "batch": 64, "groups": 4, "classes": 16, "anchors": 8400, "top": 2,
         "activation": "softmax", "dtype": "f16"},
        # rows of an open vocabulary of classes, some of them masked out, odd sizes
        {"name": "vocabulary_rows", "op": "rows", "rows": 511, "classes": 32001, "top": 10, "activation": "softmax", "dtype": "bf16",
         "masked": 0.1},
        # two rows over a very long axis
        {"name": "vocabulary_long", "op": "rows", "rows": 2, "classes": 200001, "top": 20, "activation": "softmax", "dtype": "f32",
         "masked": 0.0},
        # weights of a network's widest 1x1 convolution, quantised as they are loaded and read back
        {"name": "quantize_weights", "op": "quantize", "rows": 640, "k": 2560, "dtype": "f32"},
        # a feature map of a batch of 64 in rows of channels
        {"name": "quantize_features", "op": "quantize", "rows": 409600, "k": 320, "dtype": "f16"},
        # one row through a classifier's last layer
        {"name": "linear_row", "op": "linear", "m": 1, "k": 1280, "n": 1000, "bias": True, "act": "", "dtype": "bf16", "packed": False},
        # rows already quantised against wide weights: the largest product
        {"name": "linear_wide", "op": "linear", "m": 8192, "k": 2560, "n": 2560, "bias": True, "act": "", "dtype": "bf16", "packed": True},
        # 1x1 convolutions with folded batch norm and SiLU: one image's deepest level
        {"name": "conv_image", "op": "pointwise", "batch": 1, "k": 640, "n": 640, "h": 20, "w": 20, "act": "silu", "dtype": "f16"},
        # odd sizes: channels that end inside a block, pixels that fill no tile
        {"name": "conv_odd", "op": "pointwise", "batch": 3, "k": 400, "n": 75, "h": 37, "w": 53, "act": "silu", "dtype": "f32"},
        # the widest concatenation of a batch of 64 at stride 8
        {"name": "conv_batch", "op": "pointwise", "batch": 64, "k": 1280, "n": 320, "h": 80, "w": 80, "act": "silu", "dtype": "f16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["detections", "planes", "rows", "quantize", "linear", "pointwise"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if kind == "detections":
        gh, gw = rng.randint(5, 40), rng.randint(5, 40)      # grid of the coarsest level: inputs of 160 to 1280
        nc = _log_int(rng, 1, 400)
        anchors = 21 * gh * gw
        batch = _log_int(rng, 1, max(1, min(64, 64 * 84 * 8400 // ((4 + nc) * anchors))))
        return {"op": kind, "batch": batch, "nc": nc, "nm": rng.choice([0, 32]), "anchors": anchors, "rows": _log_int(rng, 1, 300),
                "top": rng.randint(1, min(nc, 10)), "activation": rng.choice(["none", "sigmoid", "softmax"]), "dtype": dtype}
    if kind == "planes":
        classes = _log_int(rng, 2, 100)
        anchors = 21 * rng.randint(5, 40) * rng.randint(5, 40)
        batch = _log_int(rng, 1, max(1, min(64, 64 * 4 * 16 * 8400 // (4 * classes * anchors))))
        return {"op": kind, "batch": batch, "groups": rng.randint(1, 4), "classes": classes, "anchors": anchors,
                "top": rng.randint(1, min(classes, 4)), "activation": rng.choice(["softmax", "sigmoid"]), "dtype": dtype}
    if kind == "rows":
        classes = _log_int(rng, 1, 200001)
        return {"op": kind, "rows": _log_int(rng, 1, max(1, min(4096, (1 << 24) // classes))), "classes": classes,
                "top": rng.randint(1, min(classes, 32)), "activation": rng.choice(["softmax", "softmax", "sigmoid"]), "dtype": dtype,
                "masked": rng.choice([0.0, 0.1, 0.9])}
    if kind == "quantize":
        k = _log_int(rng, 1, 4096)
        return {"op": kind, "rows": _log_int(rng, 1, (1 << 27) // k), "k": k, "dtype": dtype}
    if kind == "linear":
        k, n = _log_int(rng, 1, 4096), _log_int(rng, 1, 4096)
        return {"op": kind, "m": _log_int(rng, 1, max(1, min(1 << 15, (1 << 35) // (k * n)))), "k": k, "n": n,
                "bias": rng.random() < 0.5, "act": rng.choice(["", "silu"]), "dtype": dtype, "packed": rng.random() < 0.3}
    k, n = _log_int(rng, 8, 2560), _log_int(rng, 1, 640)
    h, w = _log_int(rng, 1, 160), _log_int(rng, 1, 160)
    return {"op": kind, "batch": _log_int(rng, 1, max(1, min(64, (1 << 28) // (h * w * (k + n))))), "k": k, "n": n, "h": h, "w": w,
            "act": rng.choice(["", "silu"]), "dtype": dtype}


# -------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    return _inputs(case, seed)


def _inputs(case, seed, raw=False):
    """What a program has in hand: weights (and rows that come packed) quantised already; with `raw`, as they were before."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def randint(hi, *shape):
        return torch.randint(0, hi, shape, generator=gen, device="cuda")

    st = {"case": case}
    op = case["op"]
    if op == "detections":
        b, nc, a, m = case["batch"], case["nc"], case["anchors"], case["rows"]
        head = randn(b, 4 + nc + case["nm"], a)
        if case["activation"] == "none":        # sigmoid scores, most of them near zero, as a trained head emits them
            head[:, 4:4 + nc] = torch.sigmoid(head[:, 4:4 + nc] * 2 - 5)
        st["head"] = head.to(dt)
        st["index"] = torch.stack([torch.randperm(a, generator=gen, device="cuda")[:m] for _ in range(b)]).to(torch.int32)
        st["count"] = (m // 2 + randint(m - m // 2 + 1, b)).to(torch.int32)
        det = randn(b, m, 6 + case["nm"])       # rows as the suppression leaves them: the class is the sixth column
        det[:, :, 5] = randint(nc, b, m).float()
        st["det"] = det
        k = case["top"]
        st["out"] = {"logprob": torch.zeros(b, m, device="cuda"), "entropy": torch.zeros(b, m, device="cuda"),
                     "top_logprob": torch.zeros(b, m, k, device="cuda"),
                     "top_index": torch.zeros(b, m, k, dtype=torch.int32, device="cuda")}
    elif op == "planes":
        b, g, c, a = case["batch"], case["groups"], case["classes"], case["anchors"]
        st["x"] = (randn(b, g * c, a) * 2).to(dt)
        st["labels"] = randint(c, b, g, a)
    elif op == "rows":
        r, c = case["rows"], case["classes"]
        x = randn(r, c) * 3
        if case["masked"]:
            x.masked_fill_(torch.rand(r, c, generator=gen, device="cuda") < case["masked"], float("-inf"))
        st["x"] = x.to(dt)
        st["labels"] = randint(c, r)
    elif op == "quantize":
        st["x"] = _features(randn(case["rows"], case["k"])).to(dt)
    else:
        k, n = case["k"], case["n"]
        weight = randn(n, k) / math.sqrt(k)
        if raw:
            st["raw_weight"] = weight
        st["bias"] = randn(n) * 0.1 if case.get("bias", True) else None
        if op == "linear":
            x = _features(randn(case["m"], k)).to(dt)
        else:
            x = _features(randn(case["batch"], k, case["h"], case["w"])).to(dt)
        if raw:
            st["x"] = x
        elif own:         # weights are quantised once, when the network is loaded; so are rows that come packed
            from object_detectors_amd import hip_ops
            st["weight"] = hip_ops.mx_quantize(weight)
            st["x"] = hip_ops.mx_quantize(x) if case.get("packed") else x
        else:
            st["weight"] = _mx_values(weight)
            st["x"] = _mx_values(x.float()) if case.get("packed") else x
    return st


def _features(x):
    """Activations after a SiLU: a long positive tail, many small negative values."""
    return x * torch.sigmoid(x) * 2


# --------------------------------------------------------------------------------------------------------- plain
def _mx_values(x):
    """MXFP4 along the last dimension, as the values it stands for (fp32): per block of 32 the scale 2^(floor(log2 max) - 2),
    elements rounded to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to the even code)."""
    k = x.shape[-1]
    pad = -k % BLOCK
    v = torch.nn.functional.pad(x.float(), (0, pad)).unflatten(-1, (-1, BLOCK))
    exponent = torch.frexp(v.abs().amax(-1, keepdim=True))[1] - 3
    scale = torch.ldexp(torch.ones_like(v[..., :1]), exponent.clamp(min=-126))
    a = (v / scale).abs()
    q = torch.where(a < 2, torch.round(a * 2) / 2, torch.where(a < 4, torch.round(a), torch.round(a / 2) * 2)).clamp(max=6)
    return (torch.copysign(q, v) * scale).flatten(-2)[..., :k]


def _silu(y, act):
    return y / (1 + torch.exp(-y)) if act == "silu" else y


def _evidence(x, labels, top, activation):
    """log probability of `labels`, entropy, and the `top` best classes of rows x (..., C), in fp32."""
    x = x.float()
    values, index = torch.sort(x, dim=-1, descending=True, stable=True)
    values, index = values[..., :top], index[..., :top].to(torch.int32)
    if activation == "softmax":
        m = x.amax(-1, keepdim=True)
        empty = m == float("-inf")
        z = x - torch.where(empty, torch.zeros_like(m), m)
        e = torch.exp(z)
        s = e.sum(-1, keepdim=True)
        t = torch.where(e > 0, e * z, torch.zeros_like(e)).sum(-1, keepdim=True)
        log_s = torch.where(empty, torch.zeros_like(s), torch.log(s))
        entropy = torch.where(empty, torch.zeros_like(s), log_s - t / s).squeeze(-1)
        offset = torch.where(empty, torch.zeros_like(m), m)
        logprob = torch.gather(x, -1, labels.long().unsqueeze(-1)) - offset - log_s
        values = values - offset - log_s
    elif activation == "sigmoid":
        def logsig(u):
            return torch.minimum(u, torch.zeros_like(u)) - torch.log1p(torch.exp(-u.abs()))
        a = x.abs()
        e = torch.exp(-a)
        h = torch.log1p(e) + torch.where(e > 0, a * e, torch.zeros_like(e)) / (1 + e)
        entropy = h.sum(-1)
        logprob = logsig(torch.gather(x, -1, labels.long().unsqueeze(-1)))
        values = logsig(values)
    else:
        h = -torch.where(x > 0, x * torch.log(x), torch.zeros_like(x)) - torch.where(x < 1, (1 - x) * torch.log1p(-x), torch.zeros_like(x))
        entropy = h.sum(-1)
        logprob = torch.log(torch.gather(x, -1, labels.long().unsqueeze(-1)))
        values = torch.log(values)
    return {"logprob": logprob.squeeze(-1), "entropy": entropy, "top_logprob": values, "top_index": index}


def _rows_of(st):
    """Rows (..., C) and labels (...) of a case, and which rows count (None: all)."""
    case = st["case"]
    if case["op"] == "detections":
        nc = case["nc"]
        scores = st["head"][:, 4:4 + nc].transpose(1, 2)
        rows = torch.gather(scores, 1, st["index"].long().unsqueeze(-1).expand(-1, -1, nc))
        valid = torch.arange(case["rows"], device="cuda") < st["count"].unsqueeze(1)
        return rows, st["det"][:, :, 5], valid
    if case["op"] == "planes":
        x = st["x"].view(case["batch"], case["groups"], case["classes"], case["anchors"]).transpose(2, 3)
        return x, st["labels"], None
    return st["x"], st["labels"], None


def _plain(st):
    case = st["case"]
    if case["op"] in ("detections", "planes", "rows"):
        rows, labels, valid = _rows_of(st)
        out = _evidence(rows, labels, case["top"], case["activation"])
        if valid is not None:       # rows behind the count stay as they were (zeros)
            out = {key: torch.where(valid if v.ndim == 2 else valid.unsqueeze(-1), v, torch.zeros_like(v)) for key, v in out.items()}
        return out
    if case["op"] == "quantize":
        return _mx_values(st["x"])
    dt = DTYPES[case["dtype"]]
    if case["op"] == "linear":
        x = st["x"] if case["packed"] else _mx_values(st["x"])
        y = torch.matmul(x, st["weight"].t())
        if st["bias"] is not None:
            y = y + st["bias"]
        return _silu(y, case["act"]).to(dt)
    x = _mx_values(st["x"].flatten(2).transpose(1, 2))
    y = torch.matmul(x, st["weight"].t()).transpose(1, 2) + st["bias"].unsqueeze(1)
    return _silu(y, case["act"]).to(dt).reshape(case["batch"], case["n"], case["h"], case["w"])


def _own(st):
    from object_detectors_amd import hip_ops
    case = st["case"]
    if case["op"] == "detections":
        nc = case["nc"]
        return hip_ops.class_logprobs(st["head"][:, 4:4 + nc].transpose(1, 2), st["det"][:, :, 5], top=case["top"],
                                      activation=case["activation"], index=st["index"], count=st["count"], out=st["out"])
    if case["op"] == "planes":
        x = st["x"].view(case["batch"], case["groups"], case["classes"], case["anchors"]).transpose(2, 3)
        return hip_ops.class_logprobs(x, st["labels"], top=case["top"], activation=case["activation"])
    if case["op"] == "rows":
        return hip_ops.class_logprobs(st["x"], st["labels"], top=case["top"], activation=case["activation"])
    if case["op"] == "quantize":
        return hip_ops.mx_dequantize(hip_ops.mx_quantize(st["x"]))
    act = case["act"] or None
    if case["op"] == "linear":
        return hip_ops.mx_linear(st["x"], st["weight"], st["bias"], act=act, dtype=DTYPES[case["dtype"]])
    return hip_ops.mx_pointwise(st["x"], st["weight"], st["bias"], act=act)


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------------------------------------- work
def work(case):
    op, es = case["op"], SIZE[case["dtype"]]
    if op == "detections":
        rows = case["batch"] * (case["rows"] + case["rows"] // 2) / 2      # counts lie between half and all of the rows
        n = rows * case["nc"]
        return {"bytes": n * es + rows * (4 + 4 + 8 + 8 * case["top"]), "flops": 8 * n}
    if op in ("planes", "rows"):
        rows = case["batch"] * case["groups"] * case["anchors"] if op == "planes" else case["rows"]
        n = rows * case["classes"]
        return {"bytes": n * es + rows * (8 + 8 + 8 * case["top"]), "flops": 8 * n}
    if op == "quantize":                # read, write packed, read packed, write the values
        n = case["rows"] * case["k"]
        packed = case["rows"] * -(-case["k"] // BLOCK) * 17
        return {"bytes": n * es + 2 * packed + n * 4, "flops": 4 * n}
    k, n = case["k"], case["n"]
    m = case["m"] if op == "linear" else case["batch"] * case["h"] * case["w"]
    blocks = -(-k // BLOCK)
    x = m * blocks * 17 if case.get("packed") else m * k * es
    return {"bytes": x + n * blocks * 17 + n * 4 + m * n * es, "flops": 2 * m * n * k}


# --------------------------------------------------------------------------------------------------------- exact
_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _mx_exact(x):
    """The format's values in fp64: the exponent from the bits of the block's largest value, elements by distance to the
    eight magnitudes (of two equally near ones the one with the even code)."""
    k = x.shape[-1]
    blocks = -(-k // BLOCK)
    v = torch.zeros(*x.shape[:-1], blocks * BLOCK, dtype=torch.float64, device=x.device)
    v[..., :k] = x.double()
    v = v.view(*x.shape[:-1], blocks, BLOCK)
    largest = v.abs().max(-1, keepdim=True).values
    exponent = ((largest.view(torch.int64) >> 52) & 2047) - 1023 - 2
    scale = ((exponent.clamp(min=-127) + 1023) << 52).view(torch.float64)
    u = v.abs() / scale
    code = torch.zeros_like(u, dtype=torch.int8)
    for c in range(1, 8):
        middle = (_GRID[c - 1] + _GRID[c]) / 2
        code += ((u > middle) | ((u == middle) & (c % 2 == 0))).to(torch.int8)
    del u
    q = torch.tensor(_GRID, dtype=torch.float64, device=x.device)[code.int()]
    return (torch.where(v < 0, -q, q) * scale).reshape(*x.shape[:-1], blocks * BLOCK)[..., :k]


def exact(case, seed):
    st = _inputs(case, seed, raw=True)
    if case["op"] in ("detections", "planes", "rows"):
        rows, labels, valid = _rows_of(st)
        x = rows.double()
        top = case["top"]
        order = torch.argsort(-x, dim=-1, stable=True)[..., :top]
        if case["activation"] == "softmax":
            lp = torch.log_softmax(x, -1)
            empty = torch.isinf(x).all(-1, keepdim=True)
            lp = torch.where(empty, torch.full_like(lp, -math.inf), lp)
            h = -(lp.exp() * torch.where(torch.isinf(lp), torch.zeros_like(lp), lp)).sum(-1)
        else:
            if case["activation"] == "sigmoid":
                lp, ln = torch.nn.functional.logsigmoid(x), torch.nn.functional.logsigmoid(-x)
            else:
                lp, ln = torch.log(x), torch.log1p(-x)
            zero = torch.zeros_like(lp)
            h = -(lp.exp() * torch.where(torch.isinf(lp), zero, lp) + ln.exp() * torch.where(torch.isinf(ln), zero, ln)).sum(-1)
        out = {"logprob": lp.gather(-1, labels.long().unsqueeze(-1)).squeeze(-1), "entropy": h,
               "top_logprob": lp.gather(-1, order), "top_index": order.to(torch.int32)}
        if valid is not None:
            for key, v in out.items():
                v[~valid] = 0
        return out
    if case["op"] == "quantize":
        return _mx_exact(st["x"])
    w = _mx_exact(st["raw_weight"])
    if case["op"] == "linear":
        y = _mx_exact(st["x"]) @ w.t()
        if st["bias"] is not None:
            y += st["bias"].double()
        return torch.nn.functional.silu(y) if case["act"] else y
    out = []
    for image in st["x"]:       # image by image: fp64 copies of a whole batch would not fit beside each other
        y = w @ _mx_exact(image.flatten(1).t().contiguous()).t().contiguous() + st["bias"].double().unsqueeze(1)
        out.append((torch.nn.functional.silu(y) if case["act"] else y).view(case["n"], case["h"], case["w"]))
    return torch.stack(out)
