"""Cases of the operators around a layer's sparse product (``liteform_ae_b200.layer``).

A layer of a graph model, or of a language model with pruned weights or a sparse pattern between its tokens, is

    h = x + r,  f = rms_norm(h) * w          rows of 32, 16 or 8 bits (e4m3 with one scale per row)
    z = A f + b,  y = act(z) + h             A sparse (CSR, float32 values)

and, in training, the gradients of both.  A case names the pass (``what``), the matrix family and size, the
number of features, the types and the activation:

  norm           rms_norm with or without the residual's addition
  norm_backward  its gradients of x and w, the gradient that comes in through h added
  product        act(A B + bias) + residual
  backward       its gradients of B, of A's values and of the bias, from the kept z
  train          product and its gradients, one after the other
  layer          norm to 8 bits and the product that reads it

``run`` computes a case in its plain form, or through the package where ``own`` is set.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
EPS = 1e-6
E4M3_MAX = 448.0
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16, "e4m3": torch.float8_e4m3fn}
BYTES = {"float32": 4, "bfloat16": 2, "float16": 2, "e4m3": 1}
PER_ROW = 32                 # entries per row of "uniform"


def _norm(name, what, rows, feats, dtype, out="", residual=True):
    c = {"what": what, "rows": rows, "feats": feats, "dtype": dtype, "out": out or dtype, "residual": residual}
    return dict(c, name=name) if name else c


def _product(name, what, matrix, rows, cols, feats, dtype, out, act, residual=True):
    c = {"what": what, "matrix": matrix, "rows": rows, "cols": cols, "feats": feats, "dtype": dtype, "out": out,
         "act": act, "residual": residual}
    return dict(c, name=name) if name else c


def listed():
    m = 1 << 20
    return [
        # a single token on its way through a model: latency is all of it
        _norm("norm token", "norm", 1, 4096, "bfloat16", "e4m3"),
        # the features of a million-node graph before its 8-bit product
        _norm("norm graph 8-bit", "norm", m, 128, "bfloat16", "e4m3"),
        # as many features as classes, no size a power of two, no residual yet (a first layer)
        _norm("norm odd f32", "norm", 200_003, 47, "float32", residual=False),
        # training: a wide hidden size
        _norm("norm backward", "norm_backward", 1 << 18, 512, "bfloat16"),
        # serving: a handful of new rows against all others
        _product("product few rows", "product", "few", 16, 1 << 18, 256, "bfloat16", "bfloat16", "gelu"),
        # the headline graph at its hidden width, 16 bits
        _product("product graph bf16", "product", "powerlaw", m, m, 128, "bfloat16", "bfloat16", "relu"),
        # the same with 8-bit features
        _product("product graph 8-bit", "product", "powerlaw", m, m, 128, "e4m3", "bfloat16", "relu"),
        # the last layer of a classifier
        _product("product odd width", "product", "powerlaw", 200_003, 200_003, 47, "float32", "float32", "gelu_tanh", False),
        # a few rows of tens of thousands of entries beside short ones
        _product("product skew f16", "product", "skew", 1 << 18, 1 << 18, 256, "float16", "float16", "silu"),
        # gradients of a wide layer
        _product("backward graph bf16", "backward", "powerlaw", 1 << 18, 1 << 18, 256, "bfloat16", "bfloat16", "gelu"),
        # a training step on a small graph in 32 bits
        _product("train small f32", "train", "zipf", 16384, 16384, 32, "float32", "float32", "silu"),
        # inference: norm to 8 bits, product, activation, residual
        _product("layer uniform 8-bit", "layer", "uniform", m, m, 64, "bfloat16", "bfloat16", "silu"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    """Features multiplied (product) or touched (norm), backward passes counted twice."""
    n = case["rows"] if case["what"].startswith("norm") else _entries(case) * (2 if case["what"] in ("backward", "train") else 1)
    return n * case["feats"]


def draw(rng):
    biggest = _cost(_product(None, "product", "powerlaw", 1 << 20, 1 << 20, 128, "bfloat16", "bfloat16", "relu"))
    while True:
        what = rng.choice(["norm", "norm", "norm_backward", "product", "product", "product", "backward", "train", "layer"])
        feats = _log_int(rng, 8, 1024)
        if rng.random() < 0.6:
            feats = max(8, feats // 8 * 8)      # most programs keep feature widths even
        dtype = rng.choice(["float32", "bfloat16", "float16"])
        residual = rng.random() < 0.7
        if what.startswith("norm"):
            rows = _log_int(rng, 1, 1 << 20)
            if rng.random() < 0.3:
                feats = _log_int(rng, 1024, 8192)
            out = rng.choice([dtype, "e4m3"]) if what == "norm" else dtype
            case = _norm(None, what, rows, feats, dtype, out, residual)
            if _cost(case) <= 1 << 28:
                return case
            continue
        matrix = rng.choice(["zipf", "powerlaw", "powerlaw", "uniform", "skew", "few"])
        cols = _log_int(rng, 2048, 1 << 20)
        rows = _log_int(rng, 1, 512) if matrix == "few" else cols
        act = rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"])
        if what == "train":      # a kink's side may hang on the last bit of z
            dtype, act = "float32", rng.choice(["none", "silu", "gelu", "gelu_tanh"])
        out = dtype
        if what == "product" and rng.random() < 0.4:
            dtype, out = "e4m3", rng.choice(["float32", "bfloat16", "float16"])
        if what == "layer":
            dtype = out = rng.choice(["bfloat16", "float16"])
            if matrix == "few":
                continue
        case = _product(None, what, matrix, rows, cols, feats, dtype, out, act, residual)
        if _cost(case) <= biggest:
            return case


# ---- matrices -----------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 2 + 1)


def _lengths(case, g):
    M, K, kind = case["rows"], case["cols"], case["matrix"]
    if kind == "uniform":
        return torch.full((M,), min(PER_ROW, K), dtype=torch.int64, device=DEV)
    u = 1.0 - torch.rand(M, generator=g, device=DEV, dtype=torch.float64)
    if kind == "few":        # neighbourhoods of new rows, some of them empty
        return (u * 33).long().clamp(max=K)
    if kind == "skew":
        n = torch.randn(M, generator=g, device=DEV, dtype=torch.float64)
        lens = torch.exp(2.0 + 1.2 * n).round().long().clamp(1, K)
        heavy = min(64, max(1, M // 64))
        lens[torch.randperm(M, generator=g, device=DEV)[:heavy]] = min(100_000, K // 8)
        return lens
    mean, power, cap = (14.0, -1.0 / 1.1, 50_000) if kind == "powerlaw" else (16.0, -1.0 / 0.8, 2048)
    raw, scale = u ** power, 1.0
    for _ in range(8):       # clipping changes the mean: rescale until it settles
        deg = (raw * scale).round().clamp(1, min(cap, K))
        scale = scale * mean / deg.mean()
    return (raw * scale).round().clamp(1, min(cap, K)).long()


def _csr(case, seed):
    """(indptr int64, indices int32 ascending and distinct in a row, values float32).  The graph is the case's,
    so that every seed has as many entries; the seed numbers its rows and columns and makes the values."""
    M, K, g = case["rows"], case["cols"], _gen(0)
    lens = _lengths(case, g)
    r = torch.repeat_interleave(torch.arange(M, device=DEV), lens)
    if case["matrix"] == "powerlaw":       # popular columns are chosen more often
        weight = torch.cumsum((lens + 1).double(), 0)
        u = torch.rand(r.numel(), generator=g, device=DEV, dtype=torch.float64) * weight[-1]
        c = torch.searchsorted(weight, u, right=True).clamp_(max=K - 1)
    else:
        c = torch.randint(0, K, (r.numel(),), generator=g, device=DEV)
    keys = torch.unique(r * K + c)         # the few that were drawn twice count once
    rows = torch.div(keys, K, rounding_mode="floor")
    g = _gen(seed)
    row, col = (torch.randperm(n, generator=g, device=DEV) for n in (M, K))
    keys = torch.sort(row[rows] * K + col[keys - rows * K])[0]
    rows = torch.div(keys, K, rounding_mode="floor")
    indices = (keys - rows * K).to(torch.int32)
    indptr = torch.zeros(M + 1, dtype=torch.int64, device=DEV)
    torch.cumsum(torch.bincount(rows, minlength=M), 0, out=indptr[1:])
    lens = torch.diff(indptr).clamp(min=1)
    vals = (torch.rand(indices.numel(), generator=g, device=DEV) * 2 - 1) / lens.float().sqrt()[rows]
    return indptr, indices, vals


def _transposed(indptr, indices, K):
    """The same entries by column: (indptr, row of every entry, its place among the entries by row)."""
    rows = torch.repeat_interleave(torch.arange(indptr.numel() - 1, device=DEV), torch.diff(indptr))
    order = torch.sort(indices, stable=True)[1]
    ptr = torch.zeros(K + 1, dtype=torch.int64, device=DEV)
    torch.cumsum(torch.bincount(indices.long(), minlength=K), 0, out=ptr[1:])
    return ptr, rows[order].to(torch.int32), order.to(torch.int32)


def _randn(shape, dtype, g):
    return torch.randn(shape, generator=g, device=DEV).to(DTYPES[dtype])


# ---- one case -----------------------------------------------------------------------------------
def prepare(case, seed):
    what, M, N = case["what"], case["rows"], case["feats"]
    g = _gen(seed + 1000)
    s = dict(case)
    if what.startswith("norm"):
        s["w"] = (1.0 + 0.1 * torch.randn(N, generator=g, device=DEV)).to(DTYPES[case["dtype"]])
        s["x"] = _randn((M, N), case["dtype"], g)
        s["r"] = _randn((M, N), case["dtype"], g) if case["residual"] else None
        if what == "norm_backward":          # h and rstd as the forward pass left them
            s["rstd"] = torch.rsqrt(s["x"].float().square().mean(1) + EPS)
            s["dy"] = _randn((M, N), case["dtype"], g)
        return s
    K = case["cols"]
    s["indptr"], s["indices"], s["vals"] = _csr(case, seed)
    s["bias"] = (0.1 * torch.randn(N, generator=g, device=DEV)).to(DTYPES[case["out"]])
    s["scale"] = None
    if what == "layer":
        s["x"], s["r"] = _randn((K, N), case["dtype"], g), _randn((K, N), case["dtype"], g)
        s["w"] = (1.0 + 0.1 * torch.randn(N, generator=g, device=DEV)).to(DTYPES[case["dtype"]])
        return s
    if case["dtype"] == "e4m3":              # rows as the norm writes them: the largest of each is 448
        b = torch.randn((K, N), generator=g, device=DEV)
        s["scale"] = b.abs().amax(1) / E4M3_MAX
        q = torch.empty((K, -(-N // 16) * 16), dtype=torch.float8_e4m3fn, device=DEV)[:, :N]
        s["B"] = q.copy_((b / s["scale"][:, None]).clamp(-E4M3_MAX, E4M3_MAX))
    else:
        s["B"] = _randn((K, N), case["dtype"], g)
    s["R"] = _randn((M, N), case["out"], g) if case["residual"] else None
    if what in ("backward", "train"):
        s["indptr_t"], s["rows_t"], s["order"] = _transposed(s["indptr"], s["indices"], K)
        s["dy"] = _randn((M, N), case["out"], g)
        if what == "backward":               # z as the forward pass kept it
            s["z"] = _randn((M, N), case["out"], g)
    return s


# plain forms
def _act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        k = math.sqrt(2 / math.pi)
        t = torch.tanh(k * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * k * (1 + 3 * 0.044715 * z * z)
    return torch.ones_like(z)


def _plain_norm(x, r, w, out):
    h = x if r is None else (x.float() + r.float()).to(x.dtype)
    f = h.float()
    rstd = torch.rsqrt(f.square().mean(1) + EPS)
    y = f * rstd[:, None] * w.float()
    if out != "e4m3":
        return y.to(DTYPES[out]), None, h, rstd
    scale = y.abs().amax(1) / E4M3_MAX
    q = torch.where(scale[:, None] > 0, y / scale[:, None], torch.zeros_like(y)).clamp(-E4M3_MAX, E4M3_MAX)
    return q.to(torch.float8_e4m3fn), scale, h, rstd


def _entry_rows(indptr):
    return torch.repeat_interleave(torch.arange(indptr.numel() - 1, device=indptr.device), torch.diff(indptr))


def _plain_sum(indptr, indices, vals, B, scale):
    v = vals if scale is None else vals * scale[indices]
    z = torch.zeros((indptr.numel() - 1, B.shape[1]), device=B.device)
    return z.index_add_(0, _entry_rows(indptr), B[indices].float() * v[:, None])


def _plain_product(s, B, scale, R):
    z = _plain_sum(s["indptr"], s["indices"], s["vals"], B, scale) + s["bias"].float()
    y = _act(z, s["act"])
    return (y if R is None else y + R.float()).to(DTYPES[s["out"]]), z


def _plain_backward(s, z):
    dz = s["dy"].float() * _act_slope(z.float(), s["act"])
    dB = _plain_sum(s["indptr_t"], s["rows_t"], s["vals"][s["order"]], dz, None)
    dvals = (dz[_entry_rows(s["indptr"])] * s["B"][s["indices"]].float()).sum(1)
    return dB.to(s["B"].dtype), dvals, dz.sum(0)


def run(s):
    what = s["what"]
    if own:
        return _run_own(s)
    if what == "norm":
        y, scale, h, rstd = _plain_norm(s["x"], s["r"], s["w"], s["out"])
        return {"y": y, "scale": scale, "h": h if s["residual"] else None, "rstd": rstd}
    if what == "norm_backward":
        h, w, dy, rstd = s["x"].float(), s["w"].float(), s["dy"].float(), s["rstd"][:, None]
        n, t = h * rstd, dy * w
        dx = rstd * (t - n * (t * n).mean(1, keepdim=True))
        if s["r"] is not None:
            dx = dx + s["r"].float()
        return {"dx": dx.to(s["x"].dtype), "dw": (dy * n).sum(0)}
    if what == "layer":
        q, scale, h, _ = _plain_norm(s["x"], s["r"], s["w"], "e4m3")
        return {"h": h, "y": _plain_product(s, q, scale, h if s["residual"] else None)[0]}
    if what == "backward":
        dB, dvals, dbias = _plain_backward(s, s["z"])
        return {"dB": dB, "dvals": dvals, "dbias": dbias}
    y, z = _plain_product(s, s["B"], s["scale"], s["R"])
    if what == "product":
        return {"y": y}
    dB, dvals, dbias = _plain_backward(s, z)
    return {"y": y, "z": z, "dB": dB, "dvals": dvals, "dbias": dbias}


def _run_own(s):
    from liteform_ae_b200 import hyb, layer
    what = s["what"]
    if what == "norm":
        n = layer.rms_norm(s["x"], s["w"], residual=s["r"], eps=EPS, out_dtype=DTYPES[s["out"]])
        return {"y": n.y, "scale": n.scale, "h": n.h if s["residual"] else None, "rstd": n.rstd}
    if what == "norm_backward":
        dx, dw = layer.rms_norm_backward(s["dy"], s["x"], s["w"], s["rstd"], dh=s["r"])
        return {"dx": dx, "dw": dw}
    A = hyb.DeviceCsr(s["indptr"], s["indices"], s["vals"], (s["rows"], s["cols"]))
    if what == "layer":
        n = layer.rms_norm(s["x"], s["w"], residual=s["r"], eps=EPS, out_dtype=torch.float8_e4m3fn)
        y = layer.spmm_csr_act(A, n.y, scale=n.scale, bias=s["bias"], activation=s["act"],
                               residual=n.h if s["residual"] else None, out_dtype=DTYPES[s["out"]])
        return {"h": n.h, "y": y}
    if what == "product":
        return {"y": layer.spmm_csr_act(A, s["B"], scale=s["scale"], bias=s["bias"], activation=s["act"],
                                        residual=s["R"], out_dtype=DTYPES[s["out"]])}
    At = layer.CsrTranspose(s["indptr_t"], s["rows_t"], s["order"], (s["cols"], s["rows"]))
    if what == "backward":
        g = layer.spmm_csr_act_backward(A, At, s["B"], s["dy"], preact=s["z"], activation=s["act"])
        return {"dB": g.dB, "dvals": g.dvalues, "dbias": g.dbias}
    z = torch.empty_like(s["dy"])
    y = layer.spmm_csr_act(A, s["B"], bias=s["bias"], activation=s["act"], residual=s["R"], preact=z)
    g = layer.spmm_csr_act_backward(A, At, s["B"], s["dy"], preact=z, activation=s["act"])
    return {"y": y, "z": z, "dB": g.dB, "dvals": g.dvalues, "dbias": g.dbias}


# ---- what a pass cannot do without ------------------------------------------------------------------
def _entries(case):
    """Expected number of stored entries."""
    M, K, kind = case["rows"], case["cols"], case["matrix"]
    if kind == "skew":
        heavy = min(64, max(1, M // 64))
        return M * math.exp(2.0 + 1.2 ** 2 / 2) + heavy * min(100_000, K // 8)
    return M * {"uniform": PER_ROW, "zipf": 16, "powerlaw": 14, "few": 16}[kind]


def work(case):
    M, N, e, o = case["rows"], case["feats"], BYTES[case["dtype"]], BYTES[case["out"]]
    if case["what"] == "norm":
        return {"bytes": M * N * (e + 2 * e * case["residual"] + o) + M * (8 if case["out"] == "e4m3" else 4) + N * e, "flops": 6 * M * N}
    if case["what"] == "norm_backward":
        return {"bytes": M * N * e * (3 + case["residual"]) + M * 4 + N * (e + 4), "flops": 10 * M * N}
    K, E = case["cols"], _entries(case)
    A = E * 8 + (M + 1) * 8
    touched = K * (1 - math.exp(-E / K)) if case["matrix"] != "powerlaw" else 0.93 * K
    if case["what"] == "layer":
        norm = K * N * 4 * e       # x, r read; h written, and read again as the residual
        return {"bytes": A + norm + M * N * o + N * (e + o), "flops": 2 * E * N + 6 * K * N}
    forward = A + touched * (N * e + (4 if case["dtype"] == "e4m3" else 0)) + M * N * o * (1 + case["residual"]) + N * o
    # dy, z read; the entries by column; dB and the values' gradient written
    backward = A + touched * N * e + M * N * o * 2 + E * 8 + K * 8 + K * N * e + E * 4 + N * 4
    if case["what"] == "product":
        return {"bytes": forward, "flops": 2 * E * N}
    if case["what"] == "backward":
        return {"bytes": backward, "flops": 4 * E * N}
    return {"bytes": forward + M * N * o + backward - A - touched * N * e, "flops": 6 * E * N}


# ---- the definition in 64 bits ----------------------------------------------------------------------
def _sigmoid64(v):
    return torch.special.expit(v)


def _act64(z, act):
    """(value, derivative)"""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return z.clamp(min=0), torch.heaviside(z, torch.zeros_like(z))
    if act == "silu":
        p = _sigmoid64(z)
        return z * p, p + z * p * (1 - p)
    if act == "gelu":
        p = torch.special.ndtr(z)
        return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    c = 2 * math.sqrt(2 / math.pi)         # (1 + tanh u) / 2 is the sigmoid of 2 u
    p = _sigmoid64(c * (z + 0.044715 * z ** 3))
    return z * p, p + z * p * (1 - p) * c * (1 + 3 * 0.044715 * z ** 2)


def _matmul64(indptr, indices, vals, shape, X):
    if not indices.numel():
        return torch.zeros((shape[0], X.shape[1]), dtype=torch.float64, device=X.device)
    return torch.sparse_csr_tensor(indptr, indices.long(), vals.double(), size=shape) @ X


def _norm64(x, r, w, out):
    h = x.double() if r is None else x.double() + r.double()
    f = h.to(x.dtype).double()             # the norm is that of the sum as it is kept
    rstd = (f.pow(2).sum(1) / f.shape[1] + EPS).pow(-0.5)
    y = torch.einsum("mn,m,n->mn", f, rstd, w.double())
    if out != "e4m3":
        return y, None, h, rstd
    scale = y.abs().max(dim=1)[0] / E4M3_MAX
    return y / scale[:, None], scale, h, rstd


def exact(case, seed):
    s = prepare(case, seed)
    what = case["what"]
    if what == "norm":
        y, scale, h, rstd = _norm64(s["x"], s["r"], s["w"], s["out"])
        return {"y": y, "scale": scale, "h": h if s["residual"] else None, "rstd": rstd}
    if what == "norm_backward":
        n = s["x"].double() * s["rstd"].double()[:, None]
        t = s["dy"].double() * s["w"].double()
        along = torch.einsum("mn,mn->m", t, n) / n.shape[1]
        dx = (t - n * along[:, None]) * s["rstd"].double()[:, None]
        return {"dx": dx if s["r"] is None else dx + s["r"].double(), "dw": torch.einsum("mn,mn->n", s["dy"].double(), n)}
    shape = (case["rows"], case["cols"])
    if what == "layer":
        q, scale, h, _ = _norm64(s["x"], s["r"], s["w"], "e4m3")
        q = q.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).double()    # the product is that of the rows as they are kept
        z = _matmul64(s["indptr"], s["indices"], s["vals"], shape, q * scale[:, None]) + s["bias"].double()
        y = _act64(z, s["act"])[0]
        return {"h": h, "y": y + h.to(s["x"].dtype).double() if s["residual"] else y}
    X = s["B"].double()
    if s["scale"] is not None:
        X = X * s["scale"].double()[:, None]
    got, z = {}, s.get("z")
    if what != "backward":
        z = _matmul64(s["indptr"], s["indices"], s["vals"], shape, X) + s["bias"].double()
        y = _act64(z, s["act"])[0]
        got["y"] = y if s["R"] is None else y + s["R"].double()
        if what == "product":
            return got
        got["z"] = z
    dz = s["dy"].double() * _act64(z.double(), s["act"])[1]
    got["dB"] = _matmul64(s["indptr_t"], s["rows_t"], s["vals"][s["order"]], shape[::-1], dz)
    got["dvals"] = torch.empty(s["indices"].numel(), dtype=torch.float64, device=DEV)
    rows = torch.bucketize(torch.arange(s["indices"].numel(), device=DEV), s["indptr"][1:], right=True)
    step = max(1, (1 << 28) // case["feats"])
    for a in range(0, rows.numel(), step):
        got["dvals"][a:a + step] = torch.einsum("en,en->e", dz[rows[a:a + step]], X[s["indices"][a:a + step].long()])
    got["dbias"] = torch.einsum("mn->n", dz)
    return got
