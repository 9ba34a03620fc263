"""Refusals of the layer operators that need no GPU, the transposed pattern, and the test's own plain forms."""
import ctypes as C

import numpy as np
import pytest
import torch

import layer_reference as ref
from liteform_ae_b200 import _cabi, layer

BAD, SMALL = _cabi.LF_ERR_INVALID_ARGUMENT, _cabi.LF_ERR_WORKSPACE_TOO_SMALL
P = 4096    # stands for a device address: refused calls read nothing
F32, BF16, E4M3 = _cabi.LF_DTYPE_F32, _cabi.LF_DTYPE_BF16, _cabi.LF_DTYPE_E4M3


def norm(**kw):
    a = dict(x=P, dtype=F32, ld_x=8, res=0, ld_res=0, sum=0, ld_sum=0, w=P, wd=F32, eps=1e-6, y=P, yd=F32, ld_y=8, scale=0,
             rstd=0, rows=2, N=8)
    a.update(kw)
    return _cabi.load().lf_rms_norm(*a.values(), 0)


@pytest.mark.parametrize("kw", [dict(N=0), dict(rows=-1), dict(ld_x=7), dict(ld_y=7), dict(dtype=E4M3), dict(dtype=7),
                                dict(wd=E4M3), dict(yd=4), dict(eps=-1.0), dict(eps=float("nan")), dict(x=0), dict(w=0),
                                dict(y=0), dict(res=P, ld_res=8), dict(res=P, ld_res=7, sum=P, ld_sum=8),
                                dict(res=P, ld_res=8, sum=P, ld_sum=7), dict(yd=E4M3)])
def test_norm_refusals(kw):
    assert norm(**kw) == BAD and _cabi.load().lf_last_error()


def test_norm_of_no_rows_does_nothing():
    assert norm(rows=0, x=0, w=0, y=0) == 0


def norm_grad(**kw):
    a = dict(dy=P, ld_dy=8, h=P, ld_h=8, dtype=F32, w=P, wd=F32, rstd=P, ds=0, ld_ds=0, dx=P, ld_dx=8, dw=P, rows=2, N=8, ws=P,
             nws=1 << 20)
    a.update(kw)
    return _cabi.load().lf_rms_norm_backward(*a.values(), 0)


@pytest.mark.parametrize("kw", [dict(N=0), dict(rows=-1), dict(ld_dy=7), dict(ld_h=7), dict(ld_dx=7), dict(ds=P, ld_ds=7),
                                dict(dtype=E4M3), dict(wd=9), dict(dy=0), dict(h=0), dict(w=0), dict(rstd=0), dict(dx=0), dict(dw=0)])
def test_norm_backward_refusals(kw):
    assert norm_grad(**kw) == BAD


@pytest.mark.parametrize("kw", [dict(nws=0), dict(ws=0), dict(nws=63)])
def test_norm_backward_workspace(kw):
    assert norm_grad(**kw) == SMALL


def product(ep=None, **kw):
    a = dict(indptr=P, indices=P, data=P, order=0, r0=0, r1=2, nnz=4, B=P, bd=F32, ldb=8, scale=0, C=P, cd=F32, ldc=8, N=8,
             ep=None if ep is None else C.byref(_cabi.LfEpilogue(**ep)), ws=P, nws=1 << 30)
    a.update(kw)
    return _cabi.load().lf_spmm_csr_act(*a.values(), 0)


@pytest.mark.parametrize("kw", [dict(N=0), dict(ldb=7), dict(ldc=7), dict(ldb=1 << 30), dict(ldc=1 << 30),
                                dict(N=(1 << 22) + 1, ldb=1 << 23, ldc=1 << 23), dict(r0=-1), dict(r0=3),
                                dict(r1=1 << 31), dict(nnz=-1), dict(bd=4), dict(cd=E4M3), dict(bd=E4M3), dict(indptr=0),
                                dict(C=0), dict(indices=0), dict(B=0), dict(order=P, data=0), dict(order=P, nnz=1 << 31),
                                dict(ep=dict(activation=5)), dict(ep=dict(activation=-1)), dict(ep=dict(bias=P, bias_dtype=E4M3)),
                                dict(ep=dict(residual=P, residual_dtype=E4M3, ld_residual=8)),
                                dict(ep=dict(residual=P, residual_dtype=F32, ld_residual=7)),
                                dict(ep=dict(preact=P, ld_preact=7)), dict(ep=dict(preact=P, ld_preact=1 << 30)),
                                dict(ep=dict(residual=P, residual_dtype=F32, ld_residual=1 << 30))])
def test_product_refusals(kw):
    assert product(**kw) == BAD


@pytest.mark.parametrize("kw", [dict(ws=0), dict(nws=63)])
def test_product_workspace(kw):
    assert product(**kw) == SMALL


def test_product_workspace_off_the_grid():
    assert product(ws=P + 4) == BAD


@pytest.mark.parametrize("kw", [dict(B=P, C=P), dict(B=P, C=2 * P, ep=dict(preact=P, ld_preact=8)),
                                dict(B=P, C=2 * P, ep=dict(preact=2 * P, ld_preact=8))])
def test_product_outputs_lie_apart(kw):
    assert product(**kw) == BAD and b"must" in _cabi.load().lf_last_error()


def test_product_of_no_rows_does_nothing():
    assert product(r1=0, indptr=0, C=0) == 0


def act_grad(**kw):
    a = dict(dy=P, ld_dy=8, z=P, ld_z=8, dtype=F32, act=_cabi.LF_ACT_SILU, dz=P, ld_dz=8, db=P, rows=2, N=8, ws=P, nws=1 << 20)
    a.update(kw)
    return _cabi.load().lf_act_backward(*a.values(), 0)


@pytest.mark.parametrize("kw", [dict(N=0), dict(rows=-1), dict(dtype=E4M3), dict(act=9), dict(dz=0, db=0), dict(dy=0), dict(z=0),
                                dict(ld_dy=7), dict(ld_z=7), dict(ld_dz=7)])
def test_act_backward_refusals(kw):
    assert act_grad(**kw) == BAD


def test_act_backward_workspace():
    assert act_grad(nws=0) == SMALL and act_grad(ws=0) == SMALL


def value_grad(**kw):
    a = dict(indptr=P, indices=P, r0=0, r1=2, nnz=4, dy=P, ld_dy=8, z=P, ld_z=8, dyd=F32, act=_cabi.LF_ACT_SILU, B=P, bd=F32, ldb=8,
             N=8, dv=P)
    a.update(kw)
    return _cabi.load().lf_spmm_csr_grad_values(*a.values(), 0)


@pytest.mark.parametrize("kw", [dict(N=0), dict(N=(1 << 22) + 1, ldb=1 << 23, ld_dy=1 << 23, ld_z=1 << 23), dict(ldb=7),
                                dict(ldb=1 << 30), dict(ld_dy=7), dict(ld_z=1 << 30), dict(r0=3), dict(r0=-1), dict(nnz=-1),
                                dict(bd=E4M3), dict(dyd=E4M3), dict(act=9), dict(indptr=0), dict(indices=0), dict(dy=0), dict(B=0),
                                dict(dv=0), dict(z=0), dict(ld_z=7)])
def test_value_grad_refusals(kw):
    assert value_grad(**kw) == BAD


def test_epilogue_struct_layout():
    assert C.sizeof(_cabi.LfEpilogue) == 3 * 8 + 2 * 8 + 3 * 4 + 4


def test_workspace_queries_are_pure():
    lib = _cabi.load()
    assert lib.lf_rms_norm_backward_workspace_bytes(0, 8) == 0
    assert lib.lf_rms_norm_backward_workspace_bytes(1000, 8) >= 32
    assert lib.lf_act_backward_workspace_bytes(1000, 8) >= 32
    sizes = [lib.lf_spmm_csr_act_workspace_bytes(n, 64, BF16) for n in (0, 1, 1000, 10 ** 6, 10 ** 8)]
    assert sizes == sorted(sizes) and sizes[0] == 0


@pytest.mark.parametrize("shape,seed", [((0, 5), 0), ((5, 0), 0), ((1, 1), 1), ((7, 12), 2), ((60, 31), 3)])
def test_transposed_pattern(shape, seed):
    import scipy.sparse as sp
    rng = np.random.default_rng(seed)
    m = sp.csr_matrix((rng.random(shape) < 0.2).astype(np.float32) * rng.random(shape).astype(np.float32))
    m.sort_indices()
    t = layer.CsrTranspose.from_host(m.indptr, m.indices, m.shape, "cpu")
    want = m.T.tocsr()
    want.sort_indices()
    assert t.shape == m.shape[::-1] and t.nnz == m.nnz
    assert np.array_equal(t.indptr.numpy(), want.indptr) and np.array_equal(t.indices.numpy(), want.indices)
    assert np.array_equal(m.data[t.order.numpy()], want.data)


@pytest.mark.parametrize("name", ref.ACTS)
def test_slopes_by_differences(name):
    z = torch.linspace(-9, 9, 1801, dtype=torch.float64) + 1e-3     # clear of the kink
    d = 1e-5
    diff = (ref.act(z + d, name) - ref.act(z - d, name)) / (2 * d)
    assert float((diff - ref.slope(z, name)).abs().max()) < 1e-8


@pytest.mark.parametrize("indptr, indices, shape", [([0, 1, 3], [0, 1], (2, 4)), ([1, 1, 2], [0, 1], (2, 4)), ([0, 2], [0, 1], (2, 4)),
                                                    ([0, 3, 2], [0, 1], (2, 4)), ([0, 1, 2], [0, 4], (2, 4)), ([0, 1, 2], [-1, 0], (2, 4))])
def test_transposed_pattern_refusals(indptr, indices, shape):
    with pytest.raises(ValueError):
        layer.CsrTranspose.from_host(np.array(indptr), np.array(indices), shape, "cpu")


def views(pitch=32):
    buf = torch.zeros(40 * pitch + 64)
    return buf, lambda rows, N, ld, at: torch.as_strided(buf, (rows, N), (ld, 1), at)


def by_bytes(a, b):
    def held(t):
        return {t.data_ptr() + 4 * (i * t.stride(0) + k) for i in range(t.shape[0]) for k in range(t.shape[1])}
    return bool(held(a) & held(b))


def test_shared_memory_of_rows():
    """Against the sets of addresses, for rows at one distance and for single rows; equal where rows lie at two distances and
    apart, or one may be taken to share."""
    buf, view = views()
    rng = np.random.default_rng(0)
    for _ in range(3000):
        ld = int(rng.integers(1, 33))
        shapes = [(int(rng.integers(0, 6)), int(rng.integers(1, ld + 1)), ld, int(rng.integers(0, 200))) for _ in range(2)]
        a, b = (view(*s) for s in shapes)
        one_step = shapes[0][0] < 2 or shapes[1][0] < 2 or all(s[1] < ld for s in shapes)
        if one_step:
            assert layer._share_memory(a, b) == by_bytes(a, b) == layer._share_memory(b, a), shapes
        else:
            assert layer._share_memory(a, b) or not by_bytes(a, b), shapes
    v, w = buf[10:50], buf[49:60]
    assert layer._share_memory(v, w) and not layer._share_memory(buf[10:49], w) and not layer._share_memory(v, buf[:0])


@pytest.mark.parametrize("out, other, refused", [
    ((4, 8, 8, 16), (20, 8, 8, 0), True),          # rows 2 to 5 of it
    ((4, 8, 8, 160), (20, 8, 8, 0), False),        # behind it
    ((20, 8, 32, 8), (20, 8, 32, 0), False),       # columns beside it
    ((20, 8, 32, 7), (20, 8, 32, 0), True),        # one column in common
    ((20, 8, 32, 25), (20, 8, 32, 0), True),       # reaches into the next row
    ((1, 8, 8, 40), (20, 8, 32, 0), False),        # a row in a gap
    ((20, 8, 8, 0), (20, 8, 8, 8), True),          # the same rows, one further
    ((4, 8, 16, 0), (4, 8, 32, 0), True)])         # another distance
def test_outputs_in_inputs_are_refused(out, other, refused):
    _, view = views()
    a, b = view(*out), view(*other)
    if refused:
        with pytest.raises(ValueError):
            layer._outputs_apart([(a, "out"), (None, "preact")], [(b, "B"), (None, "bias")], {("out", "B")})
    else:
        layer._outputs_apart([(a, "out"), (None, "preact")], [(b, "B"), (None, "bias")])


def test_outputs_that_are_an_input_itself():
    _, view = views()
    a = view(5, 8, 16, 3)
    layer._outputs_apart([(a, "out")], [(view(5, 8, 16, 3), "residual")], {("out", "residual")})
    for given, may_be in (([(a, "out")], ()), ([(a, "out"), (a, "preact")], {("out", "residual")})):
        with pytest.raises(ValueError):
            layer._outputs_apart(given, [(a, "residual")], may_be)
    with pytest.raises(ValueError):
        layer._outputs_apart([(a, "out")], [(a.view(torch.int32), "residual")], {("out", "residual")})


def act_grad_as(**kw):
    a = dict(dy=P, ld_dy=8, z=P, ld_z=8, dtype=BF16, act=_cabi.LF_ACT_SILU, dz=P, dzd=F32, ld_dz=8, db=P, rows=2, N=8, ws=P, nws=1 << 20)
    a.update(kw)
    return _cabi.load().lf_act_backward_as(*a.values(), 0)


@pytest.mark.parametrize("kw", [dict(dzd=_cabi.LF_DTYPE_F16), dict(dtype=F32, dzd=BF16), dict(dzd=E4M3), dict(dzd=9), dict(ld_dz=7), dict(N=0),
                                dict(rows=-1), dict(dtype=E4M3), dict(act=9), dict(dz=0, db=0), dict(dy=0), dict(z=0)])
def test_act_backward_as_refusals(kw):
    assert act_grad_as(**kw) == BAD


def test_act_backward_as_workspace():
    assert act_grad_as(nws=0) == SMALL and act_grad_as(rows=0, db=0, dy=0, z=0, ws=0, nws=0) == 0


def test_matrices_are_kept_by_gpu(monkeypatch):
    """A matrix uploaded while one GPU is current is not handed out for another."""
    import scipy.sparse as sp
    from liteform_ae_b200 import hyb
    from liteform_ae_b200.format_matrix_market import MTX
    m = sp.csr_matrix(np.eye(3, dtype=np.float32))
    g = MTX.from_csr(m.indptr, m.indices, m.data, m.shape, "t")
    made, current = [], [0]
    monkeypatch.setattr(hyb.DeviceCsr, "from_host", staticmethod(lambda *a: made.append(str(a[4])) or (str(a[4]), len(made))))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    first = g.csr_device()
    current[0] = 1
    second = g.csr_device()
    assert first[0] == "cuda:0" and second[0] == "cuda:1"
    assert g.csr_device("cuda:0") is first and g.csr_device(torch.device("cuda", 1)) is second and g.csr_device("cuda") is second
    assert made == ["cuda:0", "cuda:1"]


def test_infer_takes_the_matrix_to_its_rows(monkeypatch):
    from liteform_ae_b200 import pipeline

    class Stop(Exception):
        pass

    class Rows:
        is_cuda, device = True, torch.device("cuda", 3)

    class Matrix:
        def csr_device(self, device):
            raise Stop(str(device))

    with pytest.raises(Stop, match="cuda:3"):
        pipeline.infer(Matrix(), Rows(), [{}])
    with pytest.raises(ValueError):
        pipeline.infer(Matrix(), torch.zeros(3, 8), [{}])


def test_first_calls_of_two_threads(monkeypatch):
    """The types are known to a call that comes at any line of another's first one."""
    import sys
    monkeypatch.setattr(layer, "_torch", lambda: torch)
    monkeypatch.setattr(layer, "_wide", {})
    monkeypatch.setattr(layer, "_any", {})
    monkeypatch.setattr(layer._code, "__defaults__", (layer._wide,))
    seen = []

    def at_line(frame, event, arg):
        if event == "line":
            sys.settrace(None)      # the other thread's call, made here
            held = [(d, dict(d)) for d in (layer._wide, layer._any)]
            seen.append(layer._code(torch.float8_e4m3fn, layer._any))
            assert layer._code(torch.float16) == _cabi.LF_DTYPE_F16
            for d, before in held:  # as it was, for the lines that follow
                d.clear()
                d.update(before)
            sys.settrace(trace)
        return at_line

    def trace(frame, event, arg):
        return at_line if frame.f_code is layer._code.__code__ else None

    sys.settrace(trace)
    try:
        assert layer._code(torch.float32) == _cabi.LF_DTYPE_F32
    finally:
        sys.settrace(None)
    assert len(seen) > 5 and set(seen) == {E4M3}


def test_tensors_that_require_a_gradient(monkeypatch):
    monkeypatch.setattr(layer, "_torch", lambda: torch)
    p, t = torch.zeros(3, requires_grad=True), torch.zeros(3)
    layer._no_graph(t, None, p.detach())
    with pytest.raises(ValueError, match="no_grad"):
        layer._no_graph(t, None, p)
    with torch.no_grad():
        layer._no_graph(t, p)


@pytest.mark.parametrize("order", [[0, 1, 2, 3], [0, 1, 2, 3, 5], [0, 1, 2, 3, -1], [0, 1, 2, 3, 3], [0, 4, 4, 3, 2]])
def test_orders_that_are_none(order):
    t = layer.CsrTranspose.from_host(np.array([0, 2, 5]), np.array([0, 3, 0, 1, 2]), (2, 4), "cpu")
    t.order = torch.tensor(order, dtype=torch.int32)
    with pytest.raises(ValueError, match="order"):
        t.validate()


def test_order_of_another_type_or_matrix():
    from liteform_ae_b200 import hyb
    t = layer.CsrTranspose.from_host(np.array([0, 2, 5]), np.array([0, 3, 0, 1, 2]), (2, 4), "cpu")
    with pytest.raises(ValueError, match="shape"):
        t.validate(hyb.DeviceCsr(torch.tensor([0, 2, 5]), torch.zeros(5, dtype=torch.int32), None, (2, 5)))
    t.order = t.order.long()
    with pytest.raises(ValueError, match="order"):
        t.validate()


R8 = dict(res=P, ld_res=8, sum=P, ld_sum=8)
EP = dict(residual=2 * P, residual_dtype=F32, ld_residual=8, bias=P, bias_dtype=F32, preact=3 * P, ld_preact=8)


@pytest.mark.parametrize("call, kw", [(norm, dict(x=P + 2)), (norm, dict(w=P + 1)), (norm, dict(y=P + 2)), (norm, dict(rstd=P + 2)),
                                      (norm, dict(yd=E4M3, scale=P + 1)), (norm, dict(R8, res=P + 2)), (norm, dict(R8, sum=P + 3)),
                                      (norm, dict(dtype=BF16, x=P + 1)), (norm_grad, dict(dy=P + 2)), (norm_grad, dict(h=P + 1)),
                                      (norm_grad, dict(w=P + 2)), (norm_grad, dict(rstd=P + 2)), (norm_grad, dict(ds=P + 2, ld_ds=8)),
                                      (norm_grad, dict(dx=P + 2)), (norm_grad, dict(dw=P + 2)), (norm_grad, dict(ws=P + 2)),
                                      (product, dict(indptr=P + 4)), (product, dict(indices=P + 2)), (product, dict(data=P + 2)),
                                      (product, dict(order=P + 2)), (product, dict(B=P + 2)), (product, dict(C=2 * P + 2)), (product, dict(scale=P + 2)),
                                      (product, dict(bd=BF16, B=P + 1)), (product, dict(C=4 * P, ep=dict(EP, bias=P + 2))),
                                      (product, dict(C=4 * P, ep=dict(EP, residual=P + 2))), (product, dict(C=4 * P, ep=dict(EP, preact=P + 2))),
                                      (act_grad, dict(dy=P + 2)), (act_grad, dict(z=P + 2)), (act_grad, dict(dz=P + 2)), (act_grad, dict(db=P + 2)),
                                      (act_grad, dict(ws=P + 2)), (act_grad_as, dict(dz=P + 2)), (act_grad_as, dict(dy=P + 1)),
                                      (value_grad, dict(indptr=P + 4)), (value_grad, dict(indices=P + 2)), (value_grad, dict(dy=P + 2)),
                                      (value_grad, dict(z=P + 2)), (value_grad, dict(B=P + 2)), (value_grad, dict(dv=P + 2))])
def test_addresses_off_their_type(call, kw):
    assert call(**(dict(dict(C=4 * P), **kw) if call is product else kw)) == BAD and b"multiple" in _cabi.load().lf_last_error()


@pytest.mark.parametrize("change", [dict(indptr=torch.int32), dict(indices=torch.int64), dict(indptr=torch.float64), dict(shape=(5, 2)), dict(shape=(3, 2))])
def test_patterns_of_other_types_or_sizes(change):
    """Refused before anything reads them as what they are not."""
    t = layer.CsrTranspose.from_host(np.array([0, 2, 5]), np.array([0, 3, 0, 1, 2]), (2, 4), "cpu")
    for name, to in change.items():
        setattr(t, name, to if name == "shape" else getattr(t, name).to(to))
    with pytest.raises(ValueError, match="ind"):
        t.validate()
