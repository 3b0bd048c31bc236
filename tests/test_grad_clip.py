"""Global gradient norm, clipping and the clipped optimizer steps.

Expected values are computed in float64.  Tolerances: the norm is the float64 norm rounded once
to float32 (2^-24 relative; the float64 sum of squares is off by far less than 2^-40), a clipped
value is the float64 product rounded once to float32 (2^-24) and, for bfloat16, once more
(2^-8 + 2^-24).  Optimizer steps are compared bit for bit with the plain step on gradients that
were clipped before."""
import math

import numpy as np
import pytest
import torch

import oracle
import pose_estimation_amd as pe
from pose_estimation_amd import _ffi, ops

INF = math.inf
U32 = 2.0 ** -24
HALF_STEP = {torch.float32: U32, torch.bfloat16: 2.0 ** -8 + U32}


# --------------------------------------------------------------------------- CPU: refusals
def test_c_entries_refuse_bad_arguments_on_the_host():
    lib = _ffi.lib()
    E, U = _ffi.PE_E_INVALID, _ffi.PE_E_UNSUPPORTED
    one = 16   # stands for a pointer: never followed, every call is refused before a launch
    assert lib.pe_grad_norm_workspace_bytes() == 2 * _ffi.PE_NORM_MAX_SHARES
    assert lib.pe_grad_norm(None, None, 1, 0, 1.0, one, one, None) == E
    assert lib.pe_grad_norm(one, one, -1, 0, 1.0, one, one, None) == E
    assert lib.pe_grad_norm(one, one, 4097, 0, 1.0, one, one, None) == E
    assert lib.pe_grad_norm(one, one, 1, 7, 1.0, one, one, None) == U
    assert lib.pe_grad_norm(one, one, 1, 0, INF, one, one, None) == E
    assert lib.pe_grad_norm(one, one, 1, 0, 1.0, None, one, None) == E
    assert lib.pe_grad_norm(one, one, 17, 0, 1.0, one, None, None) == E
    assert lib.pe_grad_norm(one, one, 1, 0, 1.0, one, 20, None) == E
    assert lib.pe_grad_clip(one, one, 1, 0, 1.0, -1.0, one, one, None) == E
    assert lib.pe_grad_clip(one, one, 1, 0, 1.0, math.nan, one, one, None) == E
    d = _ffi.ClipDesc(None, None, 1.0, -1, 0, 1.0, 0)
    import ctypes

    def adam(p=one, grad=one, desc=d, norm=one, ws=one, n=4):
        return lib.pe_adam_clip_step(p, one, one, grad, None, n, 0.9, 0.999, 1e-8, 1e-3, 1.0,
                                     None if desc is None else ctypes.addressof(desc), norm, ws,
                                     None)

    assert adam(p=None) == E and adam(grad=8) == E and adam(desc=None) == E and adam(n=-1) == E
    assert adam(norm=None) == E and adam(ws=None, n=16385) == E and adam(ws=12) == E
    for field, bad, code in (("kind", 3, U), ("grad_scale", math.nan, E), ("max_norm", -2.0, E),
                             ("max_norm", math.nan, E), ("shares", 1, E), ("shares", 5000, E)):
        b = _ffi.ClipDesc(None, None, 1.0, -1, 0, 1.0, 0)
        setattr(b, field, bad)
        assert adam(desc=b) == code, field
        assert lib.pe_sgd_clip_step(one, one, one, None, 4, 0.1, 0.9, ctypes.addressof(b), one,
                                    one, None) == code, field


@pytest.fixture
def on_cpu(monkeypatch):
    """Lets CPU tensors past the device check, so that what lies behind it is reached."""
    monkeypatch.setattr(ops, "_need_gpu", lambda *t: None)


def test_a_set_refuses_what_it_cannot_hold(on_cpu):
    a = torch.zeros(8, 6)
    for bad in ([], [a.double()], [a.half()], [a[:, :3]], [a[:, 0]], [a[0:1].expand(4, 6)],
                [a, a], [a, a[2:4]], [a.view(-1)[:20], a.view(-1)[19:]]):
        with pytest.raises(ValueError):
            ops.GradSet(bad)
    b = torch.zeros(8, 6)
    for grads, out in (([a], [b, b]), ([a], [b.bfloat16()]), ([a], [b[:7]]), ([a], [b.t()]),
                       ([a], [a.view(-1)[6:].view(7, 6)]), ([a[:4]], [a[3:7]]), ([a, b], [b, a]),
                       ([a.t()], [b.view(6, 8)])):
        with pytest.raises(ValueError):
            ops.GradSet(grads, out=out)


def test_the_cut_covers_every_element_once_in_equal_shares(on_cpu):
    rng = np.random.default_rng(5)
    for total, most in ((1, 1), (5, 5), (4097, 37), (4097, 4097), (300_000, 37), (20_000_003, 400),
                        (400_000_001, 3)):
        count = min(total, most)
        cuts = np.sort(rng.choice(total - 1, count - 1, replace=False) + 1) if count > 1 else []
        sizes = np.diff(np.concatenate([[0], cuts, [total]])).astype(int).tolist()
        spans = [((i + 1) << 36, (i + 1) << 44, n, 4 if i % 3 else 2) for i, n in enumerate(sizes)]
        s = object.__new__(ops.GradSet)
        s.device = torch.device("cpu")
        table, shares = s._cut(spans)
        raw = table.numpy().tobytes()
        rows = np.frombuffer(raw[:s._spans * 32], dtype=ops.GradSet._SPAN)
        begin = np.frombuffer(raw[s._spans * 32:], dtype=np.int32)
        assert len(begin) == shares + 1 <= 4097 and begin[0] == 0 and begin[-1] == len(rows)
        assert (np.diff(begin) >= 0).all()
        assert (rows["n"] > 0).all() and int(rows["n"].sum()) == total
        size = np.where(rows["dtype"] == _ffi.PE_DTYPE_F32, 4, 2)
        nbytes = rows["n"] * size
        weight = sum(n * e for _, _, n, e in spans) + s.START * count
        limit = max(s.MIN_SHARE, weight / 4096) + 32
        for b, e in zip(begin, begin[1:]):   # neither many bytes nor many tensors in one share
            assert int(nbytes[b:e].sum()) <= limit and (e - b - 2) * s.START <= limit
        k = 0
        for src, dst, n, esize in spans:     # in order, contiguous
            at = 0
            while at < n * esize:
                assert rows["src"][k] == src + at and rows["dst"][k] == dst + at
                assert at % 16 == 0 and size[k] == esize
                at += int(nbytes[k])
                k += 1
            assert at == n * esize


def test_entry_points_refuse_bad_options(on_cpu):
    v = torch.zeros(8)
    for kw in (dict(max_norm=-1.0), dict(max_norm=math.nan), dict(max_norm=1.0, norm_type=1.0),
               dict(skip_nonfinite=True)):
        with pytest.raises(ValueError):
            ops.adam_step(v, v, v, v, 1, **kw)
        with pytest.raises(ValueError):
            ops.sgd_step(v, v, v, 0.1, **kw)
    with pytest.raises(ValueError):
        ops.sgd_step(v, v, v, 0.1, max_norm=1.0, p_bf16=v)
    with pytest.raises(ValueError):
        ops._norm_buffers(v.device, torch.zeros(2), None, False)
    with pytest.raises(ValueError):
        ops._norm_buffers(v.device, None, torch.zeros(100, dtype=torch.uint8), True)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        pe.nn._need_gpu(v)


def test_clipping_is_off_by_default():
    t = pe.parse_config()["train_config"]
    assert t.gradient_clip_norm is None and t.skip_nonfinite_steps is False


# --------------------------------------------------------------------------- GPU
gpu = pytest.mark.gpu


def rand(gen, n, dtype=torch.float32, scale=1.0):
    return (torch.randn(n, generator=gen, device="cuda") * scale).to(dtype)


def seeded(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def norm64(tensors, kind=2.0):
    flat = torch.cat([t.reshape(-1).double().abs() for t in tensors])
    if kind == INF:
        return float(flat.max()) if flat.numel() else 0.0
    return float(flat.square().sum().sqrt())


def assert_norm(got, want):
    assert got.shape == (1,) and got.dtype == torch.float32
    if math.isfinite(want) and want < 3.4e38:
        assert abs(float(got) - want) <= U32 * want * (1 + 1e-6) + 1.5e-45, (float(got), want)
    elif math.isnan(want):
        assert math.isnan(float(got))
    else:
        assert float(got) == INF


def assert_scaled(got, src, factor):
    want = src.double() * factor
    bound = HALF_STEP[src.dtype] * want.abs() * (1 + 1e-6) + (
        2.0 ** -149 if src.dtype == torch.float32 else 2.0 ** -133)
    assert got.dtype == src.dtype and bool(((got.double() - want).abs() <= bound).all())


SETS = {
    "one": [(1, torch.float32)],
    "small": [(3, torch.float32), (17, torch.bfloat16), (1, torch.bfloat16), (64, torch.float32)],
    "empty_inside": [(0, torch.float32), (5, torch.float32), (0, torch.bfloat16)],
    "uneven": [(70_001, torch.float32), (9, torch.bfloat16), (131_073, torch.bfloat16),
               (4096, torch.float32)],
    "large": [(5_000_001, torch.float32), (3_000_003, torch.bfloat16)],
}


@gpu
@pytest.mark.parametrize("kind", [2.0, INF])
@pytest.mark.parametrize("name", sorted(SETS))
@pytest.mark.parametrize("offset", [0, 1])
def test_norm_and_clip_against_float64(name, kind, offset):
    """offset 1: every tensor starts one element past a 16-byte boundary, with guards around it."""
    gen = seeded(7)
    hold = [rand(gen, n + 16, dt, 0.01) for n, dt in SETS[name]]
    grads = [h[8 + offset:8 + offset + n] for h, (n, _) in zip(hold, SETS[name])]
    before = [h.clone() for h in hold]
    n = norm64(grads, kind)
    assert_norm(pe.grad_norm(grads, kind), n)
    assert_norm(pe.grad_norm(grads, kind, grad_scale=-0.125), 0.125 * n)
    # into other tensors, whose alignment differs
    where = [torch.full((k + 16,), 7.0, dtype=dt, device="cuda") for k, dt in SETS[name]]
    out = [w[8:8 + k] for w, (k, _) in zip(where, SETS[name])]
    s = pe.GradSet(grads, out=out)
    assert_norm(pe.clip_grads(s, 0.5 * n, kind, grad_scale=2.0), 2.0 * n)
    for o, g, w, k in zip(out, grads, where, SETS[name]):
        assert_scaled(o, g, 0.5)
        assert bool((w[:8] == 7.0).all()) and bool((w[8 + k[0]:] == 7.0).all())
    for h, b in zip(hold, before):
        assert torch.equal(h, b)
    # in place: within the limit nothing moves, past it everything does but the guards
    assert_norm(pe.clip_grads(grads, 1.5 * n, kind), n)
    for h, b in zip(hold, before):
        assert torch.equal(h, b)
    assert_norm(pe.clip_grads(grads, 0.25 * n, kind), n)
    for h, b, (k, _) in zip(hold, before, SETS[name]):
        lo, hi = 8 + offset, 8 + offset + k
        assert_scaled(h[lo:hi], b[lo:hi], 0.25)
        assert torch.equal(h[:lo], b[:lo]) and torch.equal(h[hi:], b[hi:])


@gpu
def test_many_tensors_dense_layouts_and_determinism():
    gen = seeded(3)
    grads = [rand(gen, 1 + (i * 37) % 900, torch.bfloat16 if i % 4 == 0 else torch.float32, 0.1)
             for i in range(1500)]
    grads.append(rand(gen, 2 * 8 * 5 * 7).view(2, 8, 5, 7).to(memory_format=torch.channels_last))
    grads.append(rand(gen, 60).view(5, 12).t())
    grads.append(rand(gen, 1).view(()))
    s = pe.GradSet(grads)
    assert len(s) == 1503 and s.numel == sum(g.numel() for g in grads)
    a, b = pe.grad_norm(s), pe.grad_norm(s)
    assert torch.equal(a, b)
    n = norm64(grads)
    assert_norm(a, n)
    copies = [g.clone() for g in grads]
    pe.clip_grads(s, n / 3)
    for g, c in zip(grads, copies):
        assert_scaled(g, c, 1 / 3)
    # the set reads the tensors anew
    for g in grads:
        g.zero_()
    assert float(pe.grad_norm(s)) == 0.0
    assert float(pe.clip_grads(s, 0.0)) == 0.0


@gpu
def test_float32_extremes_neither_overflow_nor_vanish():
    big = torch.full((4,), 3e38, device="cuda")
    tiny = torch.full((9,), 1e-45, device="cuda")
    assert float(pe.grad_norm([big])) == INF                # 6e38 is past float32
    pe.clip_grads([big], 1.0)
    assert_scaled(big, torch.full((4,), 0.5, device="cuda"), 1.0)
    assert_norm(pe.grad_norm([tiny]), 3 * float(tiny[0].double()))
    huge = torch.full((1 << 20,), 1e30, device="cuda")
    assert_norm(pe.grad_norm([huge], grad_scale=1e-20), 1024 * float(huge[0].double()) * float(np.float32(1e-20)))
    with pytest.raises(_ffi.PeError):
        pe.grad_norm([tiny], grad_scale=INF)


@gpu
@pytest.mark.parametrize("kind", [2.0, INF])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("value", [math.nan, -math.nan, INF, -INF])
@pytest.mark.parametrize("where", [0, 4095, 50_000])
def test_non_finite_gradients_show(kind, dtype, value, where):
    g = rand(seeded(1), 50_001, dtype)
    g[where] = value
    other = rand(seeded(2), 10)
    n = pe.clip_grads([other, g], 1.0, kind)
    assert math.isnan(float(n)) if math.isnan(value) else float(n) == INF
    assert bool(g.isnan().all()) and bool(other.isnan().all())


@gpu
def test_limits_zero_and_infinite():
    g = rand(seeded(1), 1000)
    keep = g.clone()
    assert_norm(pe.clip_grads([g], INF), norm64([keep]))
    assert torch.equal(g, keep)
    assert_norm(pe.clip_grads([g], INF, grad_scale=0.5), 0.5 * norm64([keep]))
    assert torch.equal(g, keep * 0.5)
    pe.clip_grads([g], 0.0)
    assert bool((g == 0).all())


def arenas(n, seed):
    gen = seeded(seed)
    p, m, g = rand(gen, n, scale=0.05), rand(gen, n, scale=1e-3), rand(gen, n, scale=0.3)
    return p, m, rand(gen, n, scale=1e-3).square(), g, p.bfloat16()


@gpu
@pytest.mark.parametrize("n", [1, 4, 4369, 1_000_003])
@pytest.mark.parametrize("kind", [2.0, INF])
@pytest.mark.parametrize("share", [0.4, 3.0])
def test_clipped_steps_are_the_plain_steps_on_clipped_gradients(n, kind, share):
    scale = 0.5
    p, m, v, g, b = arenas(n, n)
    limit = share * scale * norm64([g], kind)
    clipped = torch.empty_like(g)
    want_norm = pe.clip_grads(pe.GradSet([g], out=[clipped]), limit, kind, scale)
    for bf16 in (True, False):
        for opt in ("adam", "sgd"):
            a = [t.clone() for t in (p, m, v, b)]
            w = [t.clone() for t in (p, m, v, b)]
            keep = g.clone()
            kw = dict(max_norm=limit, norm_type=kind, grad_scale=scale)
            if opt == "adam":
                norm = pe.adam_step(a[0], a[1], a[2], g, 7, p_bf16=a[3] if bf16 else None, **kw)
                assert pe.adam_step(w[0], w[1], w[2], clipped, 7, p_bf16=w[3] if bf16 else None) is None
            else:
                norm = pe.sgd_step(a[0], a[1], g, 0.1, p_bf16=a[3] if bf16 else None, **kw)
                assert pe.sgd_step(w[0], w[1], clipped, 0.1, p_bf16=w[3] if bf16 else None) is None
            assert torch.equal(norm, want_norm) and torch.equal(g, keep)
            for x, y in zip(a, w):
                assert torch.equal(x, y)
            if share > 1:      # within the limit: the bits of the plain step with this scale
                w = [t.clone() for t in (p, m, v, b)]
                if opt == "adam":
                    pe.adam_step(w[0], w[1], w[2], g, 7, p_bf16=w[3] if bf16 else None,
                                 grad_scale=scale)
                else:
                    pe.sgd_step(w[0], w[1], g, 0.1, p_bf16=w[3] if bf16 else None, grad_scale=scale)
                for x, y in zip(a, w):
                    assert torch.equal(x, y)


@gpu
def test_clipped_adam_against_the_oracle():
    n = 10_007
    p, m, v, g, _ = arenas(n, 2)
    clipped = torch.empty_like(g)
    pe.clip_grads(pe.GradSet([g], out=[clipped]), 1.0)
    assert_scaled(clipped, g, 1.0 / norm64([g]))
    want = oracle.adam_step(p.cpu().numpy(), m.cpu().numpy(), v.cpu().numpy(),
                            clipped.cpu().numpy(), 1e-3, 0.9, 0.999, 1e-8, 3)
    pe.adam_step(p, m, v, g, 3, max_norm=1.0)
    for got, w in zip((p, m, v), want):
        assert np.array_equal(got.cpu().numpy(), w)


@gpu
@pytest.mark.parametrize("opt", ["adam", "sgd"])
@pytest.mark.parametrize("value", [math.nan, INF])
def test_a_non_finite_step_is_skipped_or_shows(opt, value):
    p, m, v, g, b = arenas(5003, 9)
    g[4000] = value
    keep = [t.clone() for t in (p, m, v, b)]

    def step(**kw):
        if opt == "adam":
            return pe.adam_step(p, m, v, g, 3, p_bf16=b, **kw)
        return pe.sgd_step(p, m, g, 0.1, p_bf16=b, **kw)

    assert not math.isfinite(float(step(max_norm=1.0, skip_nonfinite=True)))
    assert not math.isfinite(float(step(max_norm=INF, skip_nonfinite=True)))
    for t, k in zip((p, m, v, b), keep):
        assert torch.equal(t, k)
    g[4000] = 1.0
    step(max_norm=INF, skip_nonfinite=True)          # finite again: the step happens
    assert not torch.equal(p, keep[0]) and bool(p.isfinite().all())
    g[4000] = value
    step(max_norm=1.0)
    assert bool(p.isnan().all()) and bool(b.isnan().all())


@gpu
def test_norm_over_a_set_wider_than_the_arena():
    p, m, v, g, b = arenas(3000, 4)
    other = rand(seeded(8), 777, torch.bfloat16)
    both = pe.GradSet([g, other])
    want = [t.clone() for t in (p, m, v)]
    clipped = [torch.empty_like(g), torch.empty_like(other)]
    n = pe.clip_grads(pe.GradSet([g, other], out=clipped), 2.0)
    pe.adam_step(*want, clipped[0], 1)
    got = pe.adam_step(p, m, v, g, 1, max_norm=2.0, norm_over=both)
    assert torch.equal(got, n)
    for x, y in zip((p, m, v), want):
        assert torch.equal(x, y)


@gpu
def test_empty_gradients():
    none = torch.empty(0, device="cuda")
    assert float(pe.grad_norm([none])) == 0.0
    assert float(pe.clip_grads([none, none.bfloat16()], 1.0)) == 0.0
    e = [torch.empty(0, device="cuda") for _ in range(4)]
    assert float(pe.adam_step(*e, 1, max_norm=1.0)) == 0.0


@gpu
def test_captured_calls_and_other_streams_give_the_eager_bits():
    gen = seeded(12)
    g = [rand(gen, n) for n in (100_000, 33, 70_001)]
    out = [torch.empty_like(t) for t in g]
    p, m, v, grad, b = arenas(50_000, 5)
    s, whole = pe.GradSet(g, out=out), pe.GradSet(g + [grad])

    def work():
        return (pe.grad_norm(s), pe.clip_grads(s, 1.0),
                pe.adam_step(p, m, v, grad, 3, p_bf16=b, max_norm=0.5, norm_over=whole),
                pe.sgd_step(p, m, grad, 0.1, max_norm=0.5))

    start = [t.clone() for t in (p, m, v, b)]

    def reset(seed):
        gen = seeded(seed)
        for t in g + [grad]:
            t.copy_(rand(gen, t.numel(), scale=0.1 * seed))
        for t, k in zip((p, m, v, b), start):
            t.copy_(k)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        told = work()
    with pytest.raises(RuntimeError, match="before the capture"):
        refused = torch.cuda.CUDAGraph()
        with torch.cuda.graph(refused):
            pe.grad_norm([grad])
    torch.cuda.synchronize()
    for seed in (1, 2, 3):
        reset(seed)
        want = [t.clone() for t in work()] + [t.clone() for t in out + [p, m, v, b]]
        reset(seed)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(list(told) + out + [p, m, v, b], want):
            assert torch.equal(x, y)


@gpu
def test_given_norm_and_workspace_are_used():
    g = rand(seeded(6), 300_000)
    out, ws = torch.zeros(1, device="cuda"), torch.zeros(ops._NORM_WS + 8, dtype=torch.uint8, device="cuda")
    s = pe.GradSet(g)
    want = pe.grad_norm(s)
    assert pe.grad_norm(s, out=out, workspace=ws) is out and torch.equal(out, want)
    assert bool(ws.any())
    out.zero_()
    assert pe.clip_grads(s, INF, out=out, workspace=ws) is out and torch.equal(out, want)
    p, m, v, grad, _ = arenas(50_000, 5)
    pe.adam_step(p, m, v, grad, 1, max_norm=1.0, workspace=ws)
    with pytest.raises(_ffi.PeError):                     # between two float64
        pe.grad_norm(s, workspace=ws[4:])


@gpu
def test_tensors_past_four_gigabytes():
    """Offsets that do not fit 32 bits, in a set and in the arenas of a step."""
    n = (1 << 31) + 5
    g = torch.zeros(n, device="cuda")
    at = torch.tensor([0, 1, n // 2, n - 2, n - 1], device="cuda")
    g[at] = torch.tensor([3.0, -1.0, 2.0, 5.0, -4.0], device="cuda")
    want = math.sqrt(55.0)
    assert_norm(pe.grad_norm([g]), want)
    assert_norm(pe.clip_grads(pe.GradSet(g[3:]), 0.5 * math.sqrt(45.0)), math.sqrt(45.0))
    assert g[at].tolist() == [3.0, -1.0, 1.0, 2.5, -2.0]
    p, mom = torch.ones(n, device="cuda"), torch.zeros(n, device="cuda")
    norm = pe.sgd_step(p, mom, g, 0.5, max_norm=1e9)
    assert_norm(norm, math.sqrt(9.0 + 1.0 + 1.0 + 6.25 + 4.0))
    assert p[at].tolist() == [-0.5, 1.5, 0.5, -0.25, 2.0] and float(p[n // 2 + 1]) == 1.0
    assert int((p != 1.0).sum()) == 5


@gpu
def test_a_recorded_call_list_repeats_the_calls():
    from pose_estimation_amd import replay

    g, out = rand(seeded(3), 70_001), torch.empty(70_001, device="cuda")
    s = pe.GradSet([g], out=[out])

    def work(x):
        g.copy_(x)
        return pe.grad_norm(s), pe.clip_grads(s, 1.0)

    rec = replay.RecordedPass(work, [rand(seeded(4), 70_001)], g.device)
    for seed in (5, 6):
        x = rand(seeded(seed), 70_001)
        got = [t.clone() for t in rec(x)] + [out.clone()]
        want = list(work(x)) + [out]
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("optimizer", ["adam", "sgd"])
def test_trainer_clips_as_configured(optimizer):
    """A trainer step with the limit equals the same step on gradients clipped beforehand, and a
    limit that is never reached equals no limit."""
    def trainer(**train):
        t = pe.Trainer({"train_config": {"batch_size": 2, "optimizer": {"name": optimizer},
                                         "preprocess": {"image_resize": [64, 64]}, **train},
                        "model_config": {"layers": [1, 1, 1, 1], "head_channels": 64}})
        t.build_model(seed=3)
        return t

    plain, loose, tight = trainer(), trainer(gradient_clip_norm=1e30), trainer(gradient_clip_norm=1e-3)
    nets = [t.net for t in (plain, loose, tight)]
    batch = next(plain.get_features_labels_data(1))
    for t in (plain, loose, tight):
        t.train_step(*batch)
    assert plain.grad_norm is None
    n = norm64([nets[2].grads])
    assert n > 1e-3
    for t in (loose, tight):
        assert_norm(t.grad_norm, norm64([t.net.grads]))
    assert torch.equal(nets[0].master, nets[1].master) and torch.equal(nets[0].work, nets[1].work)
    assert not torch.equal(nets[0].master, nets[2].master)
    again = trainer()
    clipped = torch.empty_like(nets[2].grads)
    pe.clip_grads(pe.GradSet([nets[2].grads], out=[clipped]), 1e-3)
    if optimizer == "adam":
        pe.adam_step(again.net.master, again.net.opt_m, again.net.opt_v, clipped, 1, 1e-3)
    else:
        pe.sgd_step(again.net.master, again.net.opt_m, clipped, 1e-3)
    assert torch.equal(again.net.master, nets[2].master)


@gpu
def test_trainer_skips_a_step_that_is_not_finite():
    t = pe.Trainer({"train_config": {"batch_size": 2, "skip_nonfinite_steps": True,
                                     "preprocess": {"image_resize": [64, 64]}},
                    "model_config": {"layers": [1, 1, 1, 1], "head_channels": 64}})
    t.build_model(seed=3)
    features, labels = next(t.get_features_labels_data(1))
    t.train_step(features, labels)
    assert math.isfinite(float(t.grad_norm))
    keep = t.net.master.clone()
    t.net.work.fill_(math.nan)            # as if an activation had overflowed
    t.train_step(features, labels)
    assert not math.isfinite(float(t.grad_norm))
    assert torch.equal(t.net.master, keep)


@gpu
@pytest.mark.parametrize("family", ["hrnet_w32", "mobilenet_v2"])
def test_tape_graph_networks_take_the_limit(family):
    size = [64, 64]
    cfg = {"train_config": {"batch_size": 2, "gradient_clip_norm": 1e-3,
                            "preprocess": {"image_resize": size}},
           "model_config": {"backbone": family, "width": 32, "modules": [1, 1, 1], "blocks": 1,
                            "layer1_blocks": 1}}
    t = pe.Trainer(cfg)
    t.build_model(seed=3)
    before = t.net.master.clone()
    t.train_step(*next(t.get_features_labels_data(1)))
    assert_norm(t.grad_norm, norm64([t.net.grads]))
    clipped = torch.empty_like(t.net.grads)
    pe.clip_grads(pe.GradSet([t.net.grads], out=[clipped]), 1e-3)
    pe.adam_step(before, torch.zeros_like(before), torch.zeros_like(before), clipped, 1, 1e-3)
    assert torch.equal(before, t.net.master)


@gpu
def test_lists_are_taken_without_waiting_for_the_device():
    """grad_norm and clip_grads of a plain list return while work queued before them still runs;
    several lists in a row, each with a table of its own."""
    gen = seeded(14)
    lists = [[rand(gen, n + 16 * k) for n in (50_000, 7, 3001)] for k in range(6)]
    want = [norm64(g) for g in lists]
    for _ in range(2):                     # the staging memory is there
        for g in lists:
            pe.grad_norm(g), pe.clip_grads(g, INF)
    a = torch.randn(8192, 8192, device="cuda").bfloat16()
    b = torch.mm(a, a)
    torch.cuda.synchronize()
    for _ in range(300):                   # about 0.3 s
        torch.mm(a, a, out=b)
    done = torch.cuda.Event()
    done.record()
    norms = [pe.grad_norm(g) for g in lists]
    clipped = [pe.clip_grads(g, 0.5 * n) for g, n in zip(lists, want)]
    assert not done.query()
    torch.cuda.synchronize()
    for n, c, g, w in zip(norms, clipped, lists, want):
        assert_norm(n, w)
        assert_norm(c, w)
        # every element rounded by at most half a step, so the norm of the results as well
        assert abs(norm64(g) - 0.5 * w) <= 2 * U32 * w


@gpu
def test_a_recorded_call_list_repeats_calls_on_lists():
    from pose_estimation_amd import replay

    def work(x):
        g = x.clone()
        return pe.grad_norm([g, x]), pe.clip_grads([g], 1.0), g

    rec = replay.RecordedPass(work, [rand(seeded(4), 70_001)], torch.device("cuda", 0))
    for seed in (5, 6, 7):
        x = rand(seeded(seed), 70_001)
        for a, b in zip([t.clone() for t in rec(x)], work(x)):
            assert torch.equal(a, b)


def test_a_set_knows_whether_it_holds_an_arena():
    s = object.__new__(ops.GradSet)
    v = torch.zeros(100)
    at = v.data_ptr()
    s._ranges = [(at + 40, at + 80), (at + 200, at + 240)]
    for lo, hi, held in ((0, 10, False), (0, 11, True), (12, 13, True), (19, 20, True),
                         (20, 50, False), (20, 51, True), (59, 100, True), (60, 100, False),
                         (0, 100, True), (5, 5, False)):
        assert s._holds(v[lo:hi]) is held, (lo, hi)
    s._ranges = []
    assert s._holds(v) is False


@gpu
def test_a_norm_over_other_tensors_is_refused():
    """The norm a step is clipped by has the step's own gradients in it."""
    p, m, v, g, _ = arenas(3000, 4)
    other = rand(seeded(8), 3000)
    before = [t.clone() for t in (p, m, v)]
    with pytest.raises(ValueError, match="norm_over"):
        pe.adam_step(p, m, v, g, 1, max_norm=1.0, norm_over=pe.GradSet([other]))
    with pytest.raises(ValueError, match="norm_over"):
        pe.sgd_step(p, m, g, 0.1, max_norm=1.0, norm_over=pe.GradSet([other]))
    for a, b in zip((p, m, v), before):
        assert torch.equal(a, b)
    parts = pe.GradSet([other, g[1000:2000]])       # the tensors of an arena with gaps
    assert_norm(pe.sgd_step(p, m, g, 0.1, max_norm=1.0, norm_over=parts),
                norm64([other, g[1000:2000]]))
    none = torch.empty(0, device="cuda")
    assert_norm(pe.sgd_step(none, none, none, 0.1, max_norm=1.0, norm_over=pe.GradSet([other])),
                norm64([other]))


@gpu
def test_lists_under_a_default_device():
    g = [rand(seeded(15), 5000), rand(seeded(16), 9, torch.bfloat16)]
    with torch.device("cuda"):
        assert_norm(pe.grad_norm(g), norm64(g))
        assert_norm(pe.clip_grads(pe.GradSet(g), INF), norm64(g))
