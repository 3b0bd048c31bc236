"""The row norm before and after a residual block (nn.residual_norm, nn.residual_norm_bwd).

The expected values are the formulas in float64; the tolerance of every single element comes from
a running error analysis of the same formulas in float32: `R` carries a float64 value together
with a bound of what float32 arithmetic may be off by (2^-24 for each operation, 2^-24 times the
depth of the additions for a sum), and an output adds half a step of its type.  Bounds are doubled
at the end for the second-order terms that the analysis leaves out."""
import ctypes
import itertools
import math

import numpy as np
import pytest
import torch

import pose_estimation_amd as pe
from pose_estimation_amd import _ffi, nn, ops

U = 2.0 ** -24
HALF_STEP = {torch.float32: U, torch.bfloat16: 2.0 ** -8}
ROW_DEPTH = 32        # 8 in a thread, 6 butterfly steps, at most 16 waves, and the products
BF, F = torch.bfloat16, torch.float32
TYPES = {"bf16": (BF, BF), "mixed": (BF, F), "f32": (F, F)}


class R:
    """A float64 value and a bound of its float32 evaluation's error."""

    def __init__(self, v, e=None):
        self.v = v.double()
        self.e = torch.zeros_like(self.v) if e is None else e

    def _rounded(self, v, e):
        return R(v, e + U * v.abs())

    def __add__(self, o):
        return self._rounded(self.v + o.v, self.e + o.e)

    def __sub__(self, o):
        return self._rounded(self.v - o.v, self.e + o.e)

    def __mul__(self, o):
        return self._rounded(self.v * o.v, self.v.abs() * o.e + o.v.abs() * self.e + self.e * o.e)

    def mean(self):
        v = self.v.mean(-1, keepdim=True)
        e = self.e.mean(-1, keepdim=True) + (ROW_DEPTH + 2) * U * self.v.abs().mean(-1, keepdim=True)
        return R(v, e)

    def sum(self, dim, depth):
        return R(self.v.sum(dim), self.e.sum(dim) + depth * U * self.v.abs().sum(dim))

    def rstd(self, eps):
        t = self.v + eps
        low = (t - self.e - U * t).clamp(min=eps * (1 - 4 * U))
        v = t.rsqrt()
        return R(v, (low.rsqrt() - v) + 3 * U * v)

    def sigmoid(self):
        s = torch.sigmoid(self.v)
        # exp's argument is rounded (|g| steps of its relative error), exp and the reciprocal are
        # good to two steps each
        return R(s, s * (1 - s) * (2 * self.v.abs() + 8) * U + 4 * U * s + s * (1 - s) * self.e)


ONE = R(torch.ones((), dtype=torch.float64))


def const(v, like):
    return R(torch.full((), v, dtype=torch.float64, device=like.v.device))


def normalise(v, kind, eps):
    c = v - v.mean() if kind == "layer" else v
    r = (c * c).mean().rstd(eps)
    return c * r, r


def normalise_back(w, vhat, r, kind):
    t = w - vhat * (w * vhat).mean()
    if kind == "layer":
        t = t - w.mean()
    return r * t


def gate_terms(gate, act):
    if act == "none":
        return gate, const(1.0, gate)
    s = gate.sigmoid()
    one = const(1.0, gate)
    if act == "sigmoid":
        return s, s * (one - s)
    return gate * s, s * (one + gate * (one - s))


def expected(t, norm, act, eps, groups):
    """{output name: R} for the inputs t (2-D rows) in float64."""
    y, x = R(t["y"]), R(t["x"]) if t["x"] is not None else None
    gp, bp = (R(p) if p is not None else None for p in (t["post"] or (None, None)))
    gq, bq = (R(p) if p is not None else None for p in (t["pre"] or (None, None)))
    s = R(t["scale"]) if t["scale"] is not None else None
    rows = t["y"].shape[0]
    depth = -(-rows // 256) + 24         # additions behind a parameter gradient's element
    out = {}
    if t["post"] is not None:
        yhat, ry = normalise(y, norm, eps)
    else:
        yhat, ry = y, None
    a = yhat
    if gp is not None:
        a = a * gp
    if bp is not None:
        a = a + bp
    b = a * s if s is not None else a
    if t["gate"] is not None:
        gate = R(t["gate"])
        phi, slope = gate_terms(gate, act)
        if groups:
            phi_r, slope_r = (R(q.v.expand_as(gate.v).repeat_interleave(rows // groups, 0),
                                q.e.expand_as(gate.v).repeat_interleave(rows // groups, 0))
                              for q in (phi, slope))
        else:
            phi_r, slope_r = phi, slope
        b = b * phi_r
    h = b if x is None else x + b
    out["h"] = h
    if t["pre"] is not None:
        hhat, rh = normalise(h, norm, eps)
        z = hhat
        if gq is not None:
            z = z * gq
        if bq is not None:
            z = z + bq
        out["z"] = z
    if t.get("dh") is None and t.get("dz") is None:
        return out
    d = R(t["dh"]) if t["dh"] is not None else R(torch.zeros_like(t["y"]))
    if t["pre"] is not None:
        dz = R(t["dz"])
        if gq is not None:
            out["dpre_gamma"] = (dz * hhat).sum(0, depth)
        if bq is not None:
            out["dpre_beta"] = dz.sum(0, depth)
        d = d + normalise_back(dz * gq if gq is not None else dz, hhat, rh, norm)
    if x is not None:
        out["dx"] = d
    u = d * s if s is not None else d
    da = d                                # of the branch before scale and gate
    if t["gate"] is not None:
        w = u * a * slope_r
        if groups:
            w = R(w.v.view(groups, -1, w.v.shape[1]), w.e.view(groups, -1, w.v.shape[1])).sum(1, depth)
        out["dgate"] = w
        u, da = u * phi_r, da * phi_r
    # the kernel sums da*yhat and da and combines them with gamma and beta afterwards
    p1, p0 = (da * yhat).sum(0, depth), da.sum(0, depth)
    if s is not None:
        ds = p1 * gp if gp is not None else p1
        out["dscale"] = ds if bp is None else ds + p0 * bp
    if t["post"] is not None:
        if gp is not None:
            out["dpost_gamma"] = p1 * s if s is not None else p1
        if bp is not None:
            out["dpost_beta"] = p0 * s if s is not None else p0
        u = normalise_back(u * gp if gp is not None else u, yhat, ry, norm)
    out["dy"] = u
    return out


def assert_close(got, want, name):
    assert got is not None, name
    g, v = got.double().reshape(want.v.shape), want.v
    bound = 2.0 * want.e + HALF_STEP[got.dtype] * (v.abs() + 2.0 * want.e) + 1e-38
    if got.dtype == BF:
        bound = bound + U * v.abs()
    off = (g - v).abs()
    bad = ~(off <= bound)
    assert not bool(bad.any()), (name, int(bad.sum()), float(off.max()), float(bound[bad].min()))


def make(rows, C, types="bf16", post="gb", pre="gb", scale=True, gate="none", groups=0, x=True,
         seed=0, grads=True):
    gen = torch.Generator(device="cuda").manual_seed(seed + 31 * rows + C)
    yt, xt = TYPES[types]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def pair(spec):
        if spec is None:
            return None
        return (1 + 0.2 * normal(C) if "g" in spec else None, 0.2 * normal(C) if "b" in spec else None)

    t = {"y": (normal(rows, C) + 0.5 * normal(C)).to(yt), "x": normal(rows, C).to(xt) if x else None,
         "post": pair(post), "pre": pair(pre), "scale": 0.3 * normal(C) if scale else None,
         "gate": None}
    if gate == "row":
        t["gate"] = normal(rows, C).to(yt)
    elif gate == "group":
        t["gate"] = normal(groups, C).to(yt)
    elif gate == "vector":
        t["gate"] = normal(C).to(yt)
    if grads:
        t["dh"] = normal(rows, C).to(xt if x else yt)
        t["dz"] = normal(rows, C).to(yt) if pre is not None else None
    return t


def call(t, norm, act, eps=1e-6, out=None, into=None, train=True):
    kw = dict(norm=norm, post=t["post"], pre=t["pre"], scale=t["scale"], gate=t["gate"], gate_act=act)
    h, z, stats = nn.residual_norm(t["y"], t["x"], eps=eps, want_stats=train, out=out, **kw)
    res = {"h": h, "z": z}
    if train:
        res.update(nn.residual_norm_bwd(t["dh"], t["dz"], t["y"], t["x"], stats, into=into, **kw))
    return res


def check(t, norm="layer", act="none", eps=1e-6, groups=0):
    got = call(t, norm, act, eps)
    ref = dict(t)
    if t["gate"] is not None and t["gate"].dim() == 1:
        ref["gate"], groups = t["gate"].view(1, -1), 1
    want = expected(ref, norm, act, eps, groups)
    for name, w in want.items():
        assert_close(got[name], w, name)
    assert {k for k, v in got.items() if v is not None} == set(want)


# --------------------------------------------------------------------------- CPU
@pytest.fixture
def on_cpu(monkeypatch):
    """Lets CPU tensors past the device check, so that what lies behind it is reached."""
    monkeypatch.setattr(ops, "_need_gpu", lambda *t: None)
    monkeypatch.setattr(nn, "_need_gpu", lambda *t: None)


def test_forward_refuses(on_cpu):
    y, v = torch.zeros(6, 16), torch.zeros(16)
    b = y.bfloat16()
    wide = torch.zeros(6, 48)
    for args, kw in (
            ((torch.zeros(6, 8193),), {}), ((torch.zeros(6, 0),), {}), ((torch.zeros(()),), {}),
            ((y.double(),), {}), ((y.half(),), {}), ((y, b), {}), ((b, b.half()), {}),
            ((y, torch.zeros(5, 16)), {}), ((y.t(),), {}), ((torch.zeros(4, 6, 16)[:, ::2][::2][:, :2],), {}),
            ((y,), dict(norm="batch")), ((y,), dict(eps=0.0)), ((y,), dict(eps=math.inf)),
            ((y,), dict(eps=math.nan)), ((y,), dict(gate_act="sigmoid")),
            ((y,), dict(gate=y, gate_act="relu")), ((y,), dict(gate=b)),
            ((y,), dict(gate=torch.zeros(4, 16))), ((y,), dict(gate=torch.zeros(0, 16))),
            ((y,), dict(gate=torch.zeros(6, 8))), ((y,), dict(gate=torch.zeros(2, 3, 16))),
            ((y,), dict(scale=v.double())), ((y,), dict(scale=torch.zeros(15))),
            ((y,), dict(scale=torch.zeros(32)[::2])), ((y,), dict(post=(y, None))),
            ((y,), dict(pre=(None, v.bfloat16()))), ((y,), dict(out=(None, y))),
            ((y,), dict(out=(b, None))), ((y,), dict(out=(torch.zeros(5, 16), None))),
            ((y,), dict(out=(y, None))), ((y, y.clone()), dict(out=(y, None))),
            ((y,), dict(pre=(None, None), out=(torch.zeros(6, 16), b))),
            ((wide[:, :16], wide[:, 16:32]), dict(out=(wide[:, 8:24], None))),
            ((wide[:4, :16], wide[:4, 16:32]), dict(out=(wide[1:5, 16:32], None)))):
        with pytest.raises(ValueError):
            nn.residual_norm(*args, **kw)
    one = torch.zeros(6, 16)
    with pytest.raises(ValueError):
        nn.residual_norm(y, None, pre=(None, None), out=(one, one))


def test_backward_refuses(on_cpu):
    y, v = torch.zeros(6, 16), torch.zeros(16)
    stats, on, wide = torch.zeros(4, 6), (v, None), torch.zeros(40)
    for args, kw in (
            ((None, None, y, y, None), {}), ((y, y, y, y, None), {}), ((y, None, y, y, stats), dict(pre=on)),
            ((y, None, y, y, None), dict(post=on)), ((y, None, y, y, stats[:, :5]), dict(post=on)),
            ((y, None, y, y, stats.t().contiguous().t()), dict(post=on)),
            ((y, None, y, y, stats.double()), dict(post=on)),
            ((torch.zeros(5, 16), None, y, y, None), {}), ((y.bfloat16(), None, y, y, None), {}),
            ((y, y.bfloat16(), y, y, stats), dict(pre=on)),
            ((y, None, y, y, None), dict(into={"dscale": v})),
            ((y, None, y, y, stats), dict(post=on, into={"dpost_beta": v})),
            ((y, None, y, y, stats), dict(post=on, into={"dnothing": v})),
            ((y, None, y, y, stats), dict(post=on, into={"dpost_gamma": torch.zeros(15)})),
            ((y, None, y, y, stats), dict(post=(v, v), into={"dpost_gamma": v, "dpost_beta": v})),
            ((y, None, y, y, stats), dict(post=(v, v), into={"dpost_gamma": wide[:16],
                                                             "dpost_beta": wide[15:31]}))):
        with pytest.raises(ValueError):
            nn.residual_norm_bwd(*args, **kw)


def test_ops_need_gpu_tensors():
    y = torch.zeros(2, 8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        nn.residual_norm(y)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        nn.residual_norm_bwd(y, None, y, y, None)


def test_c_entries_refuse_bad_descriptions():
    lib = _ffi.lib()
    E, U_ = _ffi.PE_E_INVALID, _ffi.PE_E_UNSUPPORTED
    one = 16   # stands for a pointer: never followed, every call is refused before a launch

    def desc(**kw):
        base = dict(rows=6, C=16, y_dtype=1, x_dtype=1, norm=0, post=1, pre=1, gate_act=0, eps=1e-6,
                    gate_rows=0, ldy=16, ldx=16, ldgate=16, ldh=16, ldz=16, lddh=16, lddz=16,
                    lddy=16, lddx=16, lddgate=16)
        base.update(kw)
        return _ffi.RnormDesc(**base)

    def fwd(d, y=one, x=one, gp=one, gate=None, h=one, z=one):
        return lib.pe_rnorm_fwd(None if d is None else ctypes.addressof(d), y, x, gp, None, None, gate,
                                None, None, h, z, None, None)

    def bwd(d, dh=one, dz=one, stats=one, gate=None, dy=one, dgate=None, dgp=one, dgq=None, ws=16,
            n=1 << 30):
        return lib.pe_rnorm_bwd(None if d is None else ctypes.addressof(d), dh, dz, one, one, stats,
                                None, None, None, gate, None, dy, one, dgate, dgp, None, None, dgq,
                                None, ws, n, None)

    assert fwd(None) == E and bwd(None) == E
    for kw, code in ((dict(C=0), E), (dict(C=8193), U_), (dict(rows=-1), E), (dict(y_dtype=2), U_),
                     (dict(y_dtype=0), U_), (dict(norm=2), U_), (dict(eps=0.0), E),
                     (dict(eps=math.nan), E), (dict(gate_rows=4), E), (dict(gate_rows=-1), E),
                     (dict(gate_act=3), U_), (dict(ldy=-16), E)):
        d = desc(**kw)
        assert fwd(d) == code and bwd(d) == code, kw
        assert lib.pe_rnorm_bwd_workspace_bytes(ctypes.addressof(d)) == 0
    assert fwd(desc(), y=None) == E and fwd(desc(), h=None) == E and fwd(desc(), z=None) == E
    assert fwd(desc(post=0)) == E and fwd(desc(gate_rows=3)) == E and fwd(desc(ldh=8)) == E
    assert fwd(desc(pre=0)) == E and fwd(desc(), x=17) == E and bwd(desc(), dh=17) == E
    assert bwd(desc(), dh=None, dz=None) == E and bwd(desc(), dz=None) == E
    assert bwd(desc(), stats=None) == E and bwd(desc(), dy=None) == E and bwd(desc(lddy=8)) == E
    assert bwd(desc(gate_rows=3), gate=one) == E and bwd(desc(gate_rows=3), dgate=one) == E
    assert bwd(desc(post=0)) == E and bwd(desc(pre=0), dgq=one) == E
    many = desc(rows=6000)
    assert bwd(many, ws=None) == E and bwd(many, ws=8) == E and bwd(many, n=10) == E
    assert fwd(desc(rows=0)) == 0
    need = lib.pe_rnorm_bwd_workspace_bytes
    for rows, C, per in itertools.product((1, 7, 1000, 200_000), (1, 64, 333, 8192), (0, 1, 2)):
        if per and rows % per == 0 or not per:
            d = desc(rows=rows, C=C, gate_rows=per)
            n = need(ctypes.addressof(d))
            items = max(1100, rows // 2) if per == 2 else 1100
            assert n <= 24 * (C + 3) * (items + 64)
            assert n >= 16 * C or (rows <= 7 and per != 2)   # one workgroup needs none


def test_the_expected_values_are_those_of_automatic_differentiation():
    """The formulas behind the bounds against torch's own gradients and against differences."""
    for norm, act, groups, post, pre in (("layer", "sigmoid", 3, True, True),
                                         ("rms", "silu", 0, True, True),
                                         ("layer", "none", 0, False, True),
                                         ("rms", "sigmoid", 1, True, False)):
        gen = torch.Generator().manual_seed(4)
        rows, C, eps = 6, 11, 1e-3

        def normal(*shape):
            return torch.randn(*shape, generator=gen, dtype=torch.float64)

        leaf = {"y": normal(rows, C), "x": normal(rows, C), "scale": normal(C),
                "gate": normal(groups or rows, C), "gp": normal(C), "bp": normal(C),
                "gq": normal(C), "bq": normal(C)}
        dh, dz = normal(rows, C), normal(rows, C)

        def loss(v):
            def N(u):
                c = u - u.mean(1, keepdim=True) if norm == "layer" else u
                return c / (c.pow(2).mean(1, keepdim=True) + eps).sqrt()

            phi = {"none": lambda g: g, "sigmoid": torch.sigmoid,
                   "silu": torch.nn.functional.silu}[act](v["gate"])
            if groups:
                phi = phi.repeat_interleave(rows // groups, 0)
            a = N(v["y"]) * v["gp"] + v["bp"] if post else v["y"]
            h = v["x"] + v["scale"] * phi * a
            total = (h * dh).sum()
            return total + ((N(h) * v["gq"] + v["bq"]) * dz).sum() if pre else total

        grad_leaf = {k: v.clone().requires_grad_() for k, v in leaf.items()}
        loss(grad_leaf).backward()
        t = {"y": leaf["y"], "x": leaf["x"], "scale": leaf["scale"], "gate": leaf["gate"],
             "post": (leaf["gp"], leaf["bp"]) if post else None,
             "pre": (leaf["gq"], leaf["bq"]) if pre else None, "dh": dh, "dz": dz if pre else None}
        got = expected(t, norm, act, eps, groups)
        names = {"y": "dy", "x": "dx", "scale": "dscale", "gate": "dgate", "gp": "dpost_gamma",
                 "bp": "dpost_beta", "gq": "dpre_gamma", "bq": "dpre_beta"}
        for k, n in names.items():
            if n in got:
                torch.testing.assert_close(got[n].v, grad_leaf[k].grad, rtol=1e-10, atol=1e-12)
                step = 1e-5
                way = normal(*leaf[k].shape)
                hi, lo = (loss({**leaf, k: leaf[k] + sign * step * way}) for sign in (1, -1))
                slope = float((got[n].v * way).sum())
                assert abs(float(hi - lo) / (2 * step) - slope) <= 1e-6 * (1 + abs(slope))


# --------------------------------------------------------------------------- GPU
gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("C", [1, 2, 7, 8, 33, 64, 120, 128, 250, 256, 264, 512, 520, 1000, 1024, 2048,
                               3001, 4096, 8191, 8192])
def test_every_width_against_float64(types, norm, C):
    check(make(37, C, types), norm)


@gpu
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 31, 32, 33, 257, 1025, 5000])
@pytest.mark.parametrize("C", [24, 256, 1032])
def test_row_counts(rows, C):
    check(make(rows, C, "mixed"), "layer")


@gpu
@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("act", ["none", "sigmoid", "silu"])
@pytest.mark.parametrize("gate,rows,groups", [("row", 37, 0), ("row", 1, 0), ("vector", 70, 0),
                                              ("group", 96, 2), ("group", 99, 33),
                                              ("group", 4000, 4), ("group", 2600, 1300)])
@pytest.mark.parametrize("C", [40, 257, 1040])
def test_gates(types, act, gate, rows, groups, C):
    check(make(rows, C, types, gate=gate, groups=groups), "layer", act, groups=groups)


@gpu
@pytest.mark.parametrize("types", ["bf16", "f32"])
@pytest.mark.parametrize("rows,groups,C", [(13_000, 6500, 40), (124_002, 62_001, 9)])
def test_gate_rows_in_the_thousands(types, rows, groups, C):
    check(make(rows, C, types, gate="group", groups=groups), "rms", "sigmoid", groups=groups)


@gpu
@pytest.mark.parametrize("post", [None, "", "g", "b", "gb"])
@pytest.mark.parametrize("pre", [None, "", "g", "b", "gb"])
@pytest.mark.parametrize("scale", [False, True])
@pytest.mark.parametrize("norm", ["layer", "rms"])
def test_parts_that_are_absent(post, pre, scale, norm):
    for x in (True, False):
        for gate in ("none", "row", "group"):
            check(make(18, 72, "bf16", post, pre, scale, gate, 3, x), norm, groups=3 * (gate == "group"))


@gpu
@pytest.mark.parametrize("post", [None, "gb"])
def test_one_of_the_incoming_gradients_alone(post):
    t = make(50, 96, "mixed", post=post)
    t["dh"] = None
    check(t)
    t = make(50, 96, "mixed", post=post, pre=None)
    check(t)


@gpu
@pytest.mark.parametrize("eps", [1e-12, 1e-5, 10.0])
def test_rows_of_one_value_and_of_zeros(eps):
    t = make(8, 64, "f32")
    t["y"][1] = 0.0
    t["y"][2] = 3.0
    t["x"][3] = 0.0
    t["y"][4] = 1e-20
    if eps < 1e-6:       # a row of one value has no direction; its rounding noise is all that is left
        t["y"][2] = 0.0
    check(t, "layer", eps=eps)
    check(t, "rms", eps=eps)


@gpu
def test_gradients_against_differences():
    """The kernel's gradients against central differences of the definition in float64.  The
    differences are good to 1e-7 of the loss's terms, the kernel to the running error bound."""
    eps = 1e-3
    t = make(5, 48, "f32", gate="row")

    def loss(v):
        q = {k: v.get(k) for k in ("y", "x", "scale", "gate")}
        q.update(post=t["post"], pre=t["pre"])
        o = expected(q, "layer", "silu", eps, 0)
        return float((o["h"].v * t["dh"].double()).sum() + (o["z"].v * t["dz"].double()).sum())

    got = call(t, "layer", "silu", eps)
    want = expected(t, "layer", "silu", eps, 0)
    base = {k: t[k].double() for k in ("y", "x", "scale", "gate")}
    gen = torch.Generator(device="cuda").manual_seed(5)
    for k in base:
        way = torch.randn(base[k].shape, generator=gen, device="cuda", dtype=torch.float64)
        step = 1e-4
        hi, lo = (loss({**base, k: base[k] + s * step * way}) for s in (1, -1))
        slope = float((got["d" + k].double() * way).sum())
        slack = float((2 * want["d" + k].e * way.abs()).sum()) + U * float(
            (want["d" + k].v * way).abs().sum())
        assert abs((hi - lo) / (2 * step) - slope) <= slack + 1e-5 * (1 + abs(slope)), k


@gpu
def test_strided_rows_views_and_guards():
    t = make(60, 40, "mixed", gate="group", groups=4)
    want = call(t, "layer", "sigmoid")
    # inputs as columns of wider tensors, 4-D maps, an unaligned column offset
    for off in (8, 3):
        wide = {k: torch.full((60, 104), 9.0, dtype=t[k].dtype, device="cuda") for k in
                ("y", "x", "dh", "dz")}
        s = dict(t)
        for k, w in wide.items():
            w[:, off:off + 40] = t[k]
            s[k] = w[:, off:off + 40].view(4, 5, 3, 40) if k != "x" else \
                w.view(4, 5, 3, 104)[..., off:off + 40]
            s[k] = w.view(4, 5, 3, 104)[..., off:off + 40]
        g = torch.full((4, 120), 9.0, dtype=BF, device="cuda")
        g[:, off:off + 40] = t["gate"]
        s["gate"] = g[:, off:off + 40]
        h = torch.full((60, 104), 5.0, dtype=F, device="cuda")
        z = torch.full((60, 104), 5.0, dtype=BF, device="cuda")
        views = [v.view(4, 5, 3, 104)[..., off:off + 40] for v in (h, z)]
        got = call(s, "layer", "sigmoid", out=views)
        ref = expected(t, "layer", "sigmoid", 1e-6, 4)
        for k, w in ref.items():
            assert_close(got[k].reshape(w.v.shape), w, k)
            if off == 8:                                       # the same kernel: the same bits
                assert torch.equal(got[k].reshape(want[k].shape), want[k]), k
        for v in (h, z):
            assert bool((v[:, :off] == 5.0).all()) and bool((v[:, off + 40:] == 5.0).all())
    # side by side in one buffer: h in the columns behind x
    both = torch.zeros(60, 80, device="cuda")
    both[:, :40] = t["x"]
    h, _, _ = nn.residual_norm(t["y"], both[:, :40], out=(both[:, 40:], None))
    assert torch.equal(h, nn.residual_norm(t["y"], t["x"])[0]) and torch.equal(both[:, :40], t["x"])
    # broadcast rows of x (stride 0)
    one = torch.randn(1, 40, device="cuda")
    a = nn.residual_norm(t["y"], one.expand(60, 40), pre=t["pre"])
    b = nn.residual_norm(t["y"], one.repeat(60, 1), pre=t["pre"])
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # rows behind the last one stay as they are
    big_h, big_z = torch.full((70, 40), 5.0, device="cuda"), torch.full((70, 40), 5.0, dtype=BF, device="cuda")
    nn.residual_norm(t["y"], t["x"], pre=t["pre"], out=(big_h[:60], big_z[:60]))
    assert bool((big_h[60:] == 5.0).all()) and bool((big_z[60:] == 5.0).all())


@gpu
@pytest.mark.parametrize("C", [5, 40, 41, 2048, 2501, 8191])
@pytest.mark.parametrize("post", [None, "gb"])
def test_in_place_and_repeated_calls_give_the_same_bits(C, post):
    t = make(300, C, "bf16", post, gate="row")
    a, b = call(t, "layer", "silu"), call(t, "layer", "silu")
    for k in a:
        assert a[k] is b[k] is None or torch.equal(a[k], b[k]), k
    y, x = t["y"].clone(), t["x"].clone()
    h, z, _ = nn.residual_norm(y, x, norm="layer", post=t["post"], pre=t["pre"], scale=t["scale"],
                               gate=t["gate"], gate_act="silu", out=(x, y))
    assert h is x and z is y
    assert torch.equal(x, a["h"]) and torch.equal(y, a["z"])


@gpu
@pytest.mark.parametrize("C", [3, 44, 513, 516, 1030, 4100])
@pytest.mark.parametrize("post", [None, "gb"])
@pytest.mark.parametrize("pre", [None, "gb"])
def test_in_place_where_threads_share_channels(C, post, pre, monkeypatch):
    """Both directions at widths whose last channels belong to two threads, in two waves where a
    row takes more than one."""
    t = make(300, C, "bf16", post, pre, gate="row")
    want = call(t, "layer", "silu")
    kw = dict(norm="layer", post=t["post"], pre=t["pre"], scale=t["scale"], gate=t["gate"],
              gate_act="silu")
    stats = nn.residual_norm(t["y"], t["x"], want_stats=True, **kw)[2]
    dh, dz = t["dh"].clone(), None if pre is None else t["dz"].clone()
    dy = torch.empty_like(t["y"]) if dz is None else dz
    fresh = iter([dy, dh, torch.empty_like(t["gate"])])   # dy, dx, dgate
    with monkeypatch.context() as m:
        m.setattr(nn, "_dense_like", lambda like: next(fresh))
        got = nn.residual_norm_bwd(dh, dz, t["y"], t["x"], stats, **kw)
    for k, v in got.items():
        assert v is want[k] is None or torch.equal(v, want[k]), k
    y, x = t["y"].clone(), t["x"].clone()
    nn.residual_norm(y, x, out=(x, y if pre else None), **kw)
    assert torch.equal(x, want["h"]) and (pre is None or torch.equal(y, want["z"]))


@gpu
@pytest.mark.parametrize("C", [24, 333, 520, 1048, 4100])
@pytest.mark.parametrize("norm", ["layer", "rms"])
def test_rows_far_from_zero_and_lopsided_rows(C, norm):
    """A mean far above the spread, and rows whose first or last few channels are far from the
    rest, so that the parts of a row that are summed apart have means of their own."""
    t = make(12, C, "f32")
    t["y"][:4] += 1000.0
    t["y"][4:6, :8] += 500.0
    t["y"][6:8, -8:] += 500.0
    t["y"][8, -1] = 4000.0
    t["x"][9] -= 1000.0
    t["x"][10, -8:] += 300.0
    check(t, norm)


@gpu
@pytest.mark.parametrize("C", [56, 1048])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_non_finite_values_stay_in_their_row(C, bad):
    clean = make(40, C, "f32", gate="row")
    a = call(clean, "layer", "sigmoid")
    for k in ("y", "x", "dh", "dz", "gate"):
        t = {n: (v.clone() if isinstance(v, torch.Tensor) else v) for n, v in clean.items()}
        t[k][17, C // 2] = bad
        b = call(t, "layer", "sigmoid")
        keep = torch.arange(40, device="cuda") != 17
        for n in ("h", "z", "dx", "dy", "dgate"):
            assert torch.equal(a[n][keep], b[n][keep]), (k, n)
        rows = [n for n in ("h", "z", "dx", "dy", "dgate") if not bool(b[n][17].isfinite().all())]
        # a gate that is infinite has the value 0 or 1
        assert rows or k == "gate", k


@gpu
def test_into_overwrites_and_arena_views():
    t = make(33, 48, "bf16")
    want = call(t, "rms", "none")
    arena = torch.full((8 + 5 * 48,), 3.0, device="cuda")
    names = ["dscale", "dpost_gamma", "dpost_beta", "dpre_gamma", "dpre_beta"]
    into = {n: arena[4 + 48 * i:4 + 48 * (i + 1)] for i, n in enumerate(names)}
    got = call(t, "rms", "none", into=into)
    for n in names:
        assert got[n] is into[n] and torch.equal(got[n], want[n])
    assert bool((arena[:4] == 3.0).all()) and bool((arena[-4:] == 3.0).all())


@gpu
def test_no_rows():
    t = make(0, 40, "bf16", gate="row")
    got = call(t, "layer", "sigmoid")
    for k in ("dscale", "dpost_gamma", "dpost_beta", "dpre_gamma", "dpre_beta"):
        assert bool((got[k] == 0).all())
    assert got["h"].shape == (0, 40) and got["dgate"].shape == (0, 40)
    t = make(0, 40, "bf16", gate="group", groups=3)
    with pytest.raises(ValueError):
        nn.residual_norm(t["y"], t["x"], gate=t["gate"][:, :20])
    assert bool((call(t, "layer", "sigmoid")["dgate"] == 0).all())


@gpu
def test_more_than_two_to_the_31_elements():
    """Offsets past 32 bits: the last rows of a long tensor are those of a short one."""
    rows, C = 270_000, 8192
    y = torch.empty(rows, C, dtype=BF, device="cuda")
    x = torch.empty(rows, C, dtype=BF, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(1)
    for v in (y, x):
        v.zero_()
        v[-64:] = torch.randn(64, C, generator=gen, device="cuda").to(BF)
        v[:64] = torch.randn(64, C, generator=gen, device="cuda").to(BF)
    g = torch.rand(C, generator=gen, device="cuda")
    kw = dict(norm="rms", post=(g, None), pre=(g, None), scale=g)
    h, z, stats = nn.residual_norm(y, x, want_stats=True, **kw)
    grads = nn.residual_norm_bwd(x, y, y, x, stats, **kw)
    for part in (slice(0, 64), slice(rows - 64, rows)):
        sy, sx = y[part].contiguous(), x[part].contiguous()
        sh, sz, ss = nn.residual_norm(sy, sx, want_stats=True, **kw)
        assert torch.equal(h[part], sh) and torch.equal(z[part], sz)
        sg = nn.residual_norm_bwd(sx, sy, sy, sx, ss, **kw)
        assert torch.equal(grads["dx"][part], sg["dx"]) and torch.equal(grads["dy"][part], sg["dy"])


@gpu
def test_captured_passes_and_other_streams_give_the_eager_bits():
    t = make(777, 136, "mixed", gate="group", groups=7)
    kw = dict(norm="layer", post=t["post"], pre=t["pre"], scale=t["scale"], gate=t["gate"],
              gate_act="sigmoid")

    def work():
        return call(t, "layer", "sigmoid")

    want = work()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = work()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for k in want:
        assert torch.equal(want[k], other[k])
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        told = work()
    with torch.cuda.graph(second, pool=graph.pool()):     # two graphs, one pool
        again = nn.residual_norm(t["y"], t["x"], **kw)[0]
    for seed in (1, 2, 3):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        for k in ("y", "x", "dh", "dz", "gate"):
            t[k].copy_(torch.randn(t[k].shape, generator=gen, device="cuda"))
        want = work()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for k in want:
            assert torch.equal(told[k], want[k]), (seed, k)
        second.replay()
        torch.cuda.synchronize()
        assert torch.equal(again, want["h"])


@gpu
@pytest.mark.parametrize("rows", [3, 900])
def test_a_recorded_call_list_repeats_both_directions(rows):
    from pose_estimation_amd import replay

    t = make(rows, 72, "mixed", gate="group", groups=3)

    def work(y, x, dh, dz):
        res = call(dict(t, y=y, x=x, dh=dh, dz=dz), "layer", "sigmoid")
        return [res[k] for k in sorted(res)]

    ins = [t[k] for k in ("y", "x", "dh", "dz")]
    rec = replay.RecordedPass(work, ins, ins[0].device)
    for seed in (1, 2):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        new = [torch.randn(v.shape, generator=gen, device="cuda").to(v.dtype) for v in ins]
        got = [v.clone() for v in rec(*new)]
        for a, b in zip(got, work(*new)):
            assert torch.equal(a, b)


@gpu
def test_a_block_of_a_network_trained_with_a_clipped_norm():
    """The operators together: two residual 1x1-conv blocks on NHWC maps with row norms and a
    per-image gate, loss, backward into a gradient arena, clipped Adam; then the same step from
    the pieces (norm, clip, plain step), and its gradients against automatic differentiation."""
    B, H, W, C = 2, 6, 5, 64
    gen = torch.Generator(device="cuda").manual_seed(2)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    names = ["w0", "w1"] + [f"{p}{i}" for i in (0, 1) for p in ("gp", "bp", "gq", "bq", "s")]
    shapes = {n: (C, 1, 1, C) if n[0] == "w" else (C,) for n in names}
    n_params = sum(math.prod(s) for s in shapes.values())
    master, grads = torch.zeros(n_params, device="cuda"), torch.zeros(n_params, device="cuda")
    at, P, G = 0, {}, {}
    for n in names:
        k = math.prod(shapes[n])
        P[n], G[n] = (a[at:at + k].view(shapes[n]) for a in (master, grads))
        at += k
        P[n].copy_(normal(*shapes[n]) * (0.1 if n[0] in "wbs" else 0.2) + (n[0] == "g"))
    work = master.bfloat16()
    Wk = {n: work[(P[n].data_ptr() - master.data_ptr()) // 4:][:C * C].view(shapes[n]) for n in ("w0", "w1")}
    gate = normal(B, C).bfloat16()
    x0, target = normal(B, H, W, C).bfloat16(), normal(B, H, W, C).bfloat16()

    def kw(i):
        return dict(norm="layer", post=(P[f"gp{i}"], P[f"bp{i}"]), pre=(P[f"gq{i}"], P[f"bq{i}"]),
                    scale=P[f"s{i}"], gate=gate, gate_act="sigmoid")

    def conv(x, w):
        return nn.conv2d(x, w)

    m, v = torch.zeros_like(master), torch.zeros_like(master)
    norms = []
    for step in range(1, 4):
        y0 = conv(x0, Wk["w0"])
        h0, z0, s0 = nn.residual_norm(y0, x0, want_stats=True, **kw(0))
        y1 = conv(z0, Wk["w1"])
        h1, z1, s1 = nn.residual_norm(y1, h0, want_stats=True, **kw(1))
        dz1 = (z1.float() - target.float()).mul_(1e-2).bfloat16()
        into = lambda i: {f"d{a}_{b}": G[f"{c}{i}"] for a, b, c in (  # noqa: E731
            ("post", "gamma", "gp"), ("post", "beta", "bp"), ("pre", "gamma", "gq"),
            ("pre", "beta", "bq"))} | {"dscale": G[f"s{i}"]}
        g1 = nn.residual_norm_bwd(None, dz1, y1, h0, s1, into=into(1), **kw(1))
        nn.conv2d_bwd_weight(z0, g1["dy"], G["w1"], 1, 1, 0)
        wt = nn.transpose_weights(Wk["w1"].view(C, 1, C), torch.empty(C, 1, C, dtype=BF, device="cuda"))
        dz0 = nn.conv2d_bwd_data(g1["dy"], wt, (H, W), 1, 1, 0)
        g0 = nn.residual_norm_bwd(g1["dx"], dz0, y0, x0, s0, into=into(0), **kw(0))
        nn.conv2d_bwd_weight(x0, g0["dy"], G["w0"], 1, 1, 0)
        if step == 1:
            leaf = {n: P[n].double().requires_grad_() for n in names}

            def N(u, g, b):
                u = u - u.mean(-1, keepdim=True)
                return u / (u.square().mean(-1, keepdim=True) + 1e-6).sqrt() * g + b

            hh, zz = x0.double(), x0.double()
            for i in (0, 1):
                w = Wk[f"w{i}"].double().view(C, C) + (leaf[f"w{i}"] - leaf[f"w{i}"].detach()).view(C, C)
                a = N(zz @ w.t(), leaf[f"gp{i}"], leaf[f"bp{i}"])
                hh = hh + leaf[f"s{i}"] * torch.sigmoid(gate.double())[:, None, None] * a
                zz = N(hh, leaf[f"gq{i}"], leaf[f"bq{i}"])
            (zz * dz1.double()).sum().backward()
            # every activation on the way is rounded to bfloat16 (at most eight in a row)
            for n in names:
                e = (G[n].double() - leaf[n].grad).norm() / leaf[n].grad.norm()
                assert float(e) <= 8 * 2.0 ** -8, (n, float(e))
        tensors = [G[n] for n in names]
        n64 = float(grads.double().norm())
        limit = 0.5 * n64
        each = pe.GradSet(tensors)
        want = [a.clone() for a in (master, m, v, work)]
        out = torch.empty_like(grads)
        clip_set = pe.GradSet([grads], out=[out])
        first = pe.clip_grads(clip_set, limit)
        pe.adam_step(want[0], want[1], want[2], out, step, p_bf16=want[3])
        norm = pe.adam_step(master, m, v, grads, step, p_bf16=work, max_norm=limit, norm_over=each)
        assert abs(float(norm) - n64) <= U * n64 * 1.001 and abs(float(first) - n64) <= U * n64 * 1.001
        # the two norms differ in the order of their float64 sums alone
        for a, b in zip((master, m, v), want):
            torch.testing.assert_close(a, b, rtol=4 * U, atol=1e-12)
        norms.append(float(norm))
    assert all(np.isfinite(norms)) and bool(master.isfinite().all())


@gpu
@pytest.mark.parametrize("types", ["bf16", "f32"])
@pytest.mark.parametrize("act", ["sigmoid", "silu"])
@pytest.mark.parametrize("gate,rows,groups", [("row", 3, 0), ("group", 4, 2)])
@pytest.mark.parametrize("C", [61, 1040, 4203])
def test_slopes_of_saturated_gates(types, act, gate, rows, groups, C):
    """dgate = phi'(gate) itself (y = dh = 1, nothing else) for gates from -30 to 30, within a bound
    relative to the slope's terms s and 1 - s, which are both tiny on one side.

    exp's argument is rounded (2|g| steps of relative error with the constant's), exp, the reciprocal
    and each sum and product add at most two steps: (2|g| + 12) U in s and in 1 - s each.  The sums
    over a group's rows, in which every term is the same, are exact or rounded by one step."""
    yt = TYPES[types][0]
    g = torch.linspace(-30, 30, C, device="cuda").to(yt)
    count = groups or rows
    gates = torch.stack([g.roll(k) for k in range(count)])
    y = torch.ones(rows, C, dtype=yt, device="cuda")
    got = nn.residual_norm_bwd(torch.ones_like(y), None, y, None, None, gate=gates, gate_act=act)["dgate"]
    g64 = gates.double()
    s, c = torch.sigmoid(g64), torch.sigmoid(-g64)
    want = s * c if act == "sigmoid" else s * (1 + g64 * c)
    terms = s * c if act == "sigmoid" else s * (1 + g64.abs() * c)
    per = rows // groups if groups else 1
    bound = per * ((4 * g64.abs() + 26) * U * terms) * (1 + HALF_STEP[yt]) + HALF_STEP[yt] * per * want.abs()
    off = (got.double() - per * want).abs()
    assert bool((off <= bound).all()), float((off / bound).max())


@gpu
def test_more_gate_rows_than_a_launch_holds():
    """17 million runs of two rows, more than the workgroups of 2^32 threads: every output is that
    of the two halves called apart, and the sum over all rows is one of every row's dz.  An item's
    sum of two values is rounded once, a slice's sum and the result once more."""
    groups, C = 17_000_000, 8
    gen = torch.Generator(device="cuda").manual_seed(6)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    t = {k: normal(2 * groups, C).bfloat16() for k in ("y", "x", "dh", "dz")}
    t.update(gate=normal(groups, C).bfloat16(), scale=normal(C), post=(normal(C), normal(C)),
             pre=(normal(C), normal(C)))

    def backward(lo, hi):
        rows = {k: t[k][2 * lo:2 * hi] for k in ("y", "x", "dh", "dz")}
        kw = dict(norm="layer", post=t["post"], pre=t["pre"], scale=t["scale"], gate=t["gate"][lo:hi],
                  gate_act="sigmoid")
        stats = nn.residual_norm(rows["y"], rows["x"], want_stats=True, **kw)[2]
        return nn.residual_norm_bwd(rows["dh"], rows["dz"], rows["y"], rows["x"], stats, **kw)

    whole = backward(0, groups)
    half = groups // 2
    for lo, hi in ((0, half), (half, groups)):
        part = backward(lo, hi)
        assert torch.equal(part["dgate"], whole["dgate"][lo:hi])
        for k in ("dy", "dx"):
            assert torch.equal(part[k], whole[k][2 * lo:2 * hi]), k
    each = t["dz"].view(groups, 2, C).float().sum(1)
    want = each.sum(0, dtype=torch.float64)
    bound = 4 * U * each.abs().sum(0, dtype=torch.float64)
    assert bool(((whole["dpre_beta"].double() - want).abs() <= bound).all())
    assert float(bound.max()) < 10 and all(bool(whole[k].isfinite().all()) for k in whole)
