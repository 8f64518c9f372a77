"""CPU: argument checks of the channels-last layer operators (Context.group_norm / linear) that need no GPU -- the C entries' descriptor checks
through the workspace queries, and the binding's shape, type and stride rules."""
import ctypes as C

import pytest
import torch

from ttc import _lib


@pytest.fixture(scope="module")
def lib():
    import os
    if not os.path.exists(_lib.LIB_PATH):
        import __graft_entry__ as g
        g.build()
    return _lib.load()


@pytest.fixture
def host():
    """a Context without a device: the checks in front of the library calls"""
    c = object.__new__(_lib.Context)
    c.torch, c.device, c._h = torch, 0, None
    return c


NORM = dict(dtype=0, activation=0, n=2, rows=9, channels=16, groups=4, x_stride=144, x_pitch=16, eps=1e-5)
LIN = dict(dtype=0, activation=0, rows=9, cin=16, cout=8, x_pitch=16, w_pitch=8, res_pitch=8, dy_pitch=8, scale=1.0)


def _norm(lib, backward=0, **kw):
    nb = C.c_size_t(123)
    st = lib.ttc_group_norm_workspace(C.byref(_lib.TTCGroupNormDesc(**{**NORM, **kw})), backward, C.byref(nb))
    return st, nb.value


def _lin(lib, backward=0, **kw):
    nb = C.c_size_t(123)
    st = lib.ttc_linear_workspace(C.byref(_lib.TTCLinearDesc(**{**LIN, **kw})), backward, C.byref(nb))
    return st, nb.value


@pytest.mark.parametrize("bad", [dict(dtype=1), dict(dtype=4), dict(activation=-1), dict(activation=6), dict(n=-1), dict(n=65536), dict(rows=-1),
                                 dict(channels=0), dict(channels=4100, groups=1, x_pitch=4100), dict(groups=0), dict(groups=3), dict(x_pitch=15), dict(x_stride=-1),
                                 dict(eps=float("nan")), dict(eps=-1.0), dict(eps=float("inf")), dict(rows=1 << 60), dict(x_pitch=1 << 60),
                                 dict(x_stride=1 << 60)])
def test_group_norm_descriptor_refusals(lib, bad):
    assert _norm(lib, **bad) == (1, 0)
    assert _norm(lib, 1, **bad) == (1, 0)


def test_group_norm_descriptor_accepts(lib):
    for kw in (dict(), dict(rows=1, x_pitch=0), dict(n=1, x_stride=0), dict(channels=4096, groups=4096, x_pitch=4096), dict(eps=0.0), dict(dtype=2), dict(dtype=3)):
        assert _norm(lib, **kw)[0] == 0 and _norm(lib, 1, **kw)[0] == 0, kw
    for backward in (0, 1):
        st, nb = _norm(lib, backward, rows=1 << 20)                       # long samples need scratch memory
        assert st == 0 and nb > 0
    assert _norm(lib, n=0) == (0, 0) and _norm(lib, rows=0) == (0, 0)
    assert lib.ttc_group_norm_workspace(None, 0, C.byref(C.c_size_t())) == 1
    assert lib.ttc_group_norm_workspace(C.byref(_lib.TTCGroupNormDesc(**NORM)), 0, None) == 1
    assert lib.ttc_group_norm(None, C.byref(_lib.TTCGroupNormDesc(**NORM)), None, None, None, None, None, None, 0, None) == 1      # no context


@pytest.mark.parametrize("bad", [dict(dtype=1), dict(activation=7), dict(rows=-1), dict(rows=1 << 31), dict(cin=0), dict(cout=0), dict(cin=65537), dict(cout=65537),
                                 dict(x_pitch=15), dict(w_pitch=7), dict(x_pitch=1 << 31), dict(scale=float("inf")), dict(scale=float("nan")),
                                 dict(rows=(1 << 31) - 1, cout=65536, w_pitch=65536)])
def test_linear_descriptor_refusals(lib, bad):
    assert _lin(lib, **bad) == (1, 0)
    assert _lin(lib, 1, **bad) == (1, 0)


def test_linear_descriptor_accepts(lib):
    for kw in (dict(), dict(rows=0), dict(rows=1, x_pitch=0), dict(cin=1, w_pitch=0), dict(dtype=3, activation=5)):
        assert _lin(lib, **kw)[0] == 0, kw
    assert _lin(lib, 1)[1] > 0 and _lin(lib, 1, rows=0) == (0, 0)
    assert lib.ttc_linear(None, C.byref(_lib.TTCLinearDesc(**LIN)), None, None, None, None, None, None, None, 0, None) == 1


def test_rows_view_rules():
    """which arrays are read in place, and as what strides"""
    wide = torch.zeros(3, 5, 7, 24)
    s = wide[..., 8:24]
    for x, lead, want in ((s, 1, (5 * 7 * 24, 24)), (s, 0, (0, 24)), (wide[:, 0, :, 4:], 1, (5 * 7 * 24, 24)), (wide[0, 0, 0, :3], 0, (0, 3)),
                          (wide[:, 1:2, 2:3, :9], 1, (5 * 7 * 24, 9))):
        y, st, pitch = _lib._rows(x, lead)
        assert y is x and (st, pitch) == want
    for x, lead in ((s[:, :, ::2].transpose(1, 2), 1), (s[:, 1:4, 1:5], 1), (wide.transpose(1, 3), 1), (torch.zeros(1, 1, 1, 4).expand(2, 3, 5, 4), 1),
                    (torch.zeros(2, 3, 1).expand(2, 3, 4), 0)):
        y, st, pitch = _lib._rows(x, lead)
        assert y.is_contiguous() and y is not x and pitch == x.shape[-1]


def test_binding_refusals(host):
    x, w = torch.zeros(4, 6, 16), torch.zeros(16, 8)
    with pytest.raises(ValueError, match="cuda:0"):
        host.linear(x, w)
    with pytest.raises(ValueError, match="cuda:0"):
        host.group_norm(x)
    with pytest.raises(ValueError, match="unknown activation"):
        host._linear_desc(x, w, "softmax", 1.0, "linear")
    for bx, bw in ((x, w.t()), (x, w.half()), (x.double(), w.double()), (x.int(), w.int()), (x, torch.zeros(2, 1, 16, 8)), (torch.zeros(()), w)):
        with pytest.raises(ValueError, match="linear"):
            host._linear_desc(bx, bw, None, 1.0, "linear")
    with pytest.raises(ValueError, match=r"gamma must be \[16\]"):
        host._layer_vec(torch.ones(8), 16, "group_norm: gamma")
    with pytest.raises(ValueError, match=r"\[n, ..., channels\]"):
        host._norm_plan(x[0, 0], 4, 1e-5, None, "group_norm", 0)
    # TF kernel shape, transposed weight copied, strided weight read in place
    d, copy, wcopy, shape = host._linear_desc(x, torch.zeros(1, 1, 16, 8), "relu", 0.1, "linear")
    assert (d.rows, d.cin, d.cout, d.x_pitch, d.w_pitch, d.activation) == (24, 16, 8, 16, 8, 1) and not copy and not wcopy and shape == (4, 6, 8)
    d, copy, wcopy, _ = host._linear_desc(x, torch.zeros(16, 20)[:, 3:11], None, 1.0, "linear")
    assert d.w_pitch == 20 and not wcopy
    d, copy, wcopy, _ = host._linear_desc(x, torch.zeros(8, 16).t(), None, 1.0, "linear")
    assert d.w_pitch == 8 and wcopy
    assert host._layer_vec(torch.ones(16, dtype=torch.float64)[::2], 8, "p").dtype == torch.float32


def test_plans_are_kept_by_shape_alone_and_bounded(host):
    made = []
    for i in range(10000):
        host._layer_plan(("k", i % 5000), lambda: made.append(i) or i)
    assert len(host._plans) <= 4096
    n = len(made)
    host._layer_plan(("k", 4999), lambda: made.append(0))
    assert len(made) == n


class Recorder:
    """the library with its layer entries replaced by ones that note their descriptors: the binding's own work, without a device"""
    def __init__(self, lib):
        self.lib, self.calls = lib, []

    def __getattr__(self, name):
        if name in ("ttc_linear", "ttc_linear_backward", "ttc_group_norm", "ttc_group_norm_backward"):
            return lambda h, ref, *rest: self.calls.append((name, ref._obj, rest)) or 0
        return getattr(self.lib, name)


@pytest.fixture
def recorded(lib, host):
    host.lib, host.device, host._layer_stream = Recorder(lib), -1, lambda: 0       # tensors of the CPU are device -1
    return host


def test_numbers_given_as_tensors_are_read_at_every_call(recorded):
    x, w, dy, s = torch.zeros(4, 16), torch.zeros(16, 8), torch.zeros(4, 8), torch.tensor(0.5)
    for v in (0.5, 2.0):
        s.fill_(v)
        recorded.linear(x, w, scale=s)
        recorded.linear_backward(dy, x, w, scale=s)
        recorded.group_norm(x, groups=4, eps=s)
    assert [getattr(d, "scale", None) or d.eps for _, d, _ in recorded.lib.calls] == [0.5] * 3 + [2.0] * 3
    g = torch.tensor(4)
    for v in (4, 8):
        g.fill_(v)
        recorded.group_norm(x, groups=g)
        assert recorded.lib.calls[-1][1].groups == v
    with pytest.raises(ValueError, match="groups must be a whole number"):
        recorded.group_norm(x, groups=2.5)
    p = torch.tensor(1.0, requires_grad=True)
    for call in (lambda: recorded.linear(x, w, scale=p), lambda: recorded.linear_backward(dy, x, w, scale=p), lambda: recorded.group_norm(x, groups=4, eps=p)):
        with pytest.raises(ValueError, match="no gradient flows"):
            call()
    with torch.no_grad():
        recorded.linear(x, w, scale=p)
    assert recorded.lib.calls[-1][1].scale == 1.0


def test_forward_mode_tangents_are_refused(recorded):
    import torch.autograd.forward_ad as fw
    x, w, dy, g, st = torch.zeros(4, 16), torch.zeros(16, 8), torch.zeros(4, 8), torch.ones(16), torch.zeros(4, 4, 2)
    with fw.dual_level():
        dual = lambda a: fw.make_dual(a, torch.ones_like(a))      # noqa: E731
        for call in (lambda: recorded.linear(dual(x), w), lambda: recorded.linear(x, dual(w)), lambda: recorded.linear(x, w, residual=dual(dy)),
                     lambda: recorded.linear(x, w, bias=dual(torch.zeros(8))), lambda: recorded.group_norm(dual(x), groups=4),
                     lambda: recorded.group_norm(x, g, dual(g), groups=4), lambda: recorded.linear_backward(dual(dy), x, w),
                     lambda: recorded.group_norm_backward(x, x, dual(g), None, st)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        assert not recorded.lib.calls
        recorded.linear(x, w)                                     # no tangent: an ordinary call
        recorded.group_norm_backward(x, x, g, None, st)
    assert len(recorded.lib.calls) == 2


def test_a_left_out_bias_is_noticed_where_it_would_be_read(recorded):
    import warnings
    for cin, cout in ((16, 8), (16, 300)):                        # narrow: formed again from x, w and bias; wide: the kept preact
        x, w, dy, bias = torch.zeros(4, cin), torch.zeros(cin, cout), torch.zeros(4, cout), torch.zeros(cout)
        _, pre = recorded.linear(x, w, bias, activation="swish", want_preact=True)
        assert (pre is None) == (cout == 8)
        with warnings.catch_warnings():
            warnings.simplefilter("error")
            recorded.linear_backward(dy, x, w, pre, bias, activation="swish")
            recorded.linear_backward(dy, x, w, None, None, activation="swish")          # a layer without one
            recorded.linear_backward(dy, x, w)                                          # no activation: nothing to form
            if pre is not None:
                recorded.linear_backward(dy, x, w, pre, activation="swish")
                continue
        with pytest.warns(UserWarning, match="pass the forward call's bias"):
            recorded.linear_backward(dy, x, w, pre, activation="swish")


def test_stated_errors_of_the_polynomials():
    """the tanh series and the normal tail's fit, with the coefficients of the header, in float64 against their functions"""
    import math
    import os
    import re
    import numpy as np
    from scipy.special import erfcx
    text = open(os.path.join(os.path.dirname(_lib.__file__), "csrc", "layers_common.h")).read()
    body = re.search(r"float tanh_rel\(float v\) \{(.*?)\n\}", text, re.S).group(1)
    c = [float(a) / float(b) for a, b in re.findall(r"(-?\d+)\.0f / (\d+)", body.split("const float e")[0])]
    v = np.linspace(1e-3, 0.5, 2001)
    p = v + v * sum(k * v ** (2 * i + 2) for i, k in enumerate(c))
    assert len(c) == 7 and np.abs(p / np.tanh(v) - 1).max() < 9e-9
    body = re.search(r"float normal_tail\(float z, float\* e\) \{(.*?)\n\}", text, re.S).group(1)
    c = [float(a) for a in re.findall(r"-?0\.\d{6,}(?=f)", body.split("const float p =")[1].split(";")[0])]
    z = np.concatenate([np.linspace(0, 40, 40001), np.geomspace(40, 1e6, 2000)])
    t = 1 / (1 + 0.356 * z / math.sqrt(2))
    assert len(c) == 10 and np.abs(t * sum(k * t ** i for i, k in enumerate(c)) / (erfcx(z / math.sqrt(2)) / 2) - 1).max() < 4e-8
