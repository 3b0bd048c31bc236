"""The cases on which the gradient-norm, clipping and residual-norm operators are measured.

`listed()` holds the fixed cases, `draw()` gives more of the same ranges, `prepare()` makes a
case's inputs on the GPU, `run()` is one pass, in plain torch operations or (own = True) through
the framework's calls, `exact()` is the same in 64 bits and `work()` what a pass cannot do without.
"""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "bf16": 2}


# --------------------------------------------------------------------------- cases
def _grads(name, op, count, total, types, limit=1.0, **more):
    """Gradients of `count` tensors with `total` elements in all; limit = max_norm / norm."""
    return dict(name=name, op=op, count=count, total=total, types=types, limit=limit, **more)


def _norm(name, op, rows, ch, y="bf16", x="bf16", norm="layer", post=True, pre=True, bias=True,
          scale=True, gate="none", groups=0, act="none"):
    return dict(name=name, op=op, rows=rows, ch=ch, y=y, x=x, norm=norm, post=post, pre=pre,
                bias=bias, scale=scale, gate=gate, groups=groups, act=act)


def listed():
    return [
        # the heads of a three-label network: a handful of small tensors, where latency counts
        _grads("norm_heads", "norm", 9, 21_403, "mixed"),
        # every tensor of the ResNet-50 pose network, float32
        _grads("norm_resnet", "norm", 170, 34_000_000, "f32"),
        # clipped copies for the exchange: gradients of a MobileNetV2-sized trunk, both types
        _grads("clip_mobilenet", "clip", 52, 2_224_001, "mixed", 0.37),
        # the ResNet-50 pose network's gradients gathered per stage
        _grads("clip_resnet", "clip", 48, 34_000_000, "f32", 0.5),
        # the optimizer step of the final 1x1 convolution alone (fine-tuning a head)
        _grads("adam_head", "adam", 1, 4_369, "f32", 0.25),
        # the optimizer step of the whole ResNet-50 pose network, clipping active
        _grads("adam_resnet", "adam", 1, 34_000_000, "f32", 0.5),
        # one token of a wide residual stream, as in serving
        _norm("fwd_token", "fwd", 1, 4096, norm="rms", bias=False),
        # the reference's batch of two, 64x48 maps with 256 channels, one gate row per image
        _norm("fwd_maps", "fwd", 6144, 256, gate="group", groups=2, act="sigmoid"),
        # a long prompt over a float32 residual stream, gate per token
        _norm("fwd_stream", "fwd", 8192, 4096, x="f32", norm="rms", bias=False, gate="row",
              act="silu"),
        # an odd width in float32: no row starts on a 16-byte border
        _norm("train_odd", "train", 1217, 333, y="f32", x="f32", scale=False),
        # training, batch 64 at 64x48 maps, 256 channels, one gate row per image
        _norm("train_maps", "train", 196608, 256, gate="group", groups=64, act="sigmoid"),
        # training, the last stage's 2048 channels at 12x9 maps, batch 32, float32 residual
        _norm("train_deep", "train", 3456, 2048, x="f32", norm="rms", bias=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "clip", "adam", "fwd", "fwd", "train", "train"])
    if op in ("norm", "clip", "adam"):
        total = _log(rng, 1_000, 34_000_000)
        count = 1 if op == "adam" else min(_log(rng, 1, 170 if op == "norm" else 48), total)
        c = _grads("", op, count, total, "f32" if op == "adam" else rng.choice(["f32", "bf16", "mixed"]),
                   round(rng.choice([rng.uniform(0.1, 0.9), rng.uniform(1.1, 3.0)]), 3))
    else:
        # from 8 channels: with one or two the normalised row is a sign and its gradient vanishes
        ch = rng.choice([_log(rng, 8, 8192), 8 * _log(rng, 1, 1024)])
        rows = _log(rng, 1, max(2, min(200_000, 33_000_000 // ch)))
        y, x = rng.choice([("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32")])
        post, pre = rng.choice([(True, True), (True, False), (False, True)])
        gate = rng.choice(["none", "group", "row"])
        groups = 0
        if gate == "group":
            groups = min(_log(rng, 1, 64), rows)
            rows -= rows % groups
        c = _norm("", op, rows, ch, y, x, rng.choice(["layer", "rms"]), post, pre,
                  rng.random() < 0.5, rng.random() < 0.5, gate, groups,
                  rng.choice(["none", "sigmoid", "silu"]) if gate != "none" else "none")
    del c["name"]
    return c


# --------------------------------------------------------------------------- inputs
def _lengths(count, total, seed):
    """`count` positive lengths that sum to `total`, spread over about three decades."""
    g = torch.Generator().manual_seed(seed)
    w = torch.exp(torch.rand(count, generator=g, dtype=torch.float64) * 7.0)
    n = torch.clamp((w / w.sum() * (total - count)).floor().long(), min=0) + 1
    n[0] += total - int(n.sum())
    return n.tolist()


def _gradient_types(case):
    kinds = {"f32": ["f32"], "bf16": ["bf16"], "mixed": ["f32", "bf16", "f32"]}[case["types"]]
    return [kinds[i % len(kinds)] for i in range(case["count"])]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    s = {"case": case}
    if case["op"] in ("norm", "clip", "adam"):
        lengths = _lengths(case["count"], case["total"], case["count"] + case["total"])
        flat = normal(case["total"])
        parts = list(flat.split(lengths))
        sizes = torch.exp(normal(case["count"])).tolist()          # layers differ in magnitude
        s["grads"] = [(p * (1e-3 * a)).to(_DTYPES[t])
                      for p, a, t in zip(parts, sizes, _gradient_types(case))]
        # what such a run would use: a limit near the norm that these gradients have
        expect = 1e-3 * math.sqrt(sum(n * a * a for n, a in zip(lengths, sizes)))
        s["max_norm"] = case["limit"] * expect
        if case["op"] == "clip":
            s["out"] = [torch.empty_like(g) for g in s["grads"]]
        if case["op"] == "adam":
            n = case["total"]
            s["p"], s["m"] = normal(n) * 0.02, normal(n) * 1e-4
            s["v"] = normal(n).square() * 1e-6
            s["p_bf16"] = s["p"].to(torch.bfloat16)
            s["step"] = 100
        if own:
            from pose_estimation_amd import ops

            if case["op"] != "adam":
                s["set"] = ops.GradSet(s["grads"], out=s.get("out"))
        return s
    rows, ch, yt, xt = case["rows"], case["ch"], _DTYPES[case["y"]], _DTYPES[case["x"]]
    loud = 1.0 + 3.0 * torch.rand(ch, generator=gen, device="cuda").square()
    s["y"] = (normal(rows, ch) + 0.3 * normal(ch)).to(yt)
    s["x"] = (normal(rows, ch) * loud).to(xt)
    for part in ("post", "pre"):
        if case[part]:
            beta = 0.1 * normal(ch) if case["bias"] else None
            s[part] = (1.0 + 0.1 * normal(ch), beta)
        else:
            s[part] = None
    s["scale"] = 0.1 + 0.05 * normal(ch) if case["scale"] else None
    s["gate"] = None
    if case["gate"] != "none":
        s["gate"] = normal(case["groups"] if case["gate"] == "group" else rows, ch).to(yt)
    if case["op"] == "train":
        s["dh"] = (normal(rows, ch) * 1e-3).to(xt)
        s["dz"] = (normal(rows, ch) * 1e-3).to(yt) if case["pre"] else None
    return s


# --------------------------------------------------------------------------- plain forms
_BETA1, _BETA2, _ADAM_EPS, _LR, _EPS = 0.9, 0.999, 1e-8, 1e-3, 1e-6


def _plain_norm(grads):
    flat = torch.cat([g.reshape(-1).float() for g in grads])
    return flat.square().sum(dtype=torch.float64).sqrt()


def _plain_factor(norm, limit):
    return torch.where(norm > limit, limit / norm, torch.ones_like(norm)).float()


def _phi(g, act):
    if act == "none":
        return g
    sig = 1.0 / (1.0 + torch.exp(-g))
    return sig if act == "sigmoid" else g * sig


def _dphi(g, act):
    if act == "none":
        return torch.ones_like(g)
    sig = 1.0 / (1.0 + torch.exp(-g))
    return sig * (1.0 - sig) if act == "sigmoid" else sig * (1.0 + g * (1.0 - sig))


def _normalise(v, kind):
    if kind == "layer":
        v = v - v.mean(dim=1, keepdim=True)
    rstd = torch.rsqrt(v.square().mean(dim=1, keepdim=True) + _EPS)
    return v * rstd, rstd


def _normalise_back(w, vhat, rstd, kind):
    t = w - vhat * (w * vhat).mean(dim=1, keepdim=True)
    if kind == "layer":
        t = t - w.mean(dim=1, keepdim=True)
    return t * rstd


def _affine(vhat, gb):
    t = vhat * gb[0]
    return t if gb[1] is None else t + gb[1]


def _plain_forward(s):
    case = s["case"]
    y, kind = s["y"].float(), case["norm"]
    k = {}
    if s["post"] is not None:
        k["yhat"], k["yr"] = _normalise(y, kind)
        a = _affine(k["yhat"], s["post"])
    else:
        k["yhat"], a = y, y
    b = a if s["scale"] is None else a * s["scale"]
    if s["gate"] is not None:
        phi = _phi(s["gate"].float(), case["act"])
        if case["gate"] == "group":
            phi = phi.repeat_interleave(case["rows"] // case["groups"], dim=0)
        k["phi"] = phi
        b = b * phi
    h = s["x"].float() + b
    z = None
    if s["pre"] is not None:
        k["hhat"], k["hr"] = _normalise(h, kind)
        z = _affine(k["hhat"], s["pre"]).to(s["y"].dtype)
    k["a"] = a
    return h.to(s["x"].dtype), z, k


def _plain_backward(s, k):
    case, kind = s["case"], s["case"]["norm"]
    out = {}
    d = s["dh"].float()
    if s["pre"] is not None:
        dz = s["dz"].float()
        out["dpre_gamma"] = (dz * k["hhat"]).sum(dim=0)
        if s["pre"][1] is not None:
            out["dpre_beta"] = dz.sum(dim=0)
        d = d + _normalise_back(dz * s["pre"][0], k["hhat"], k["hr"], kind)
    out["dx"] = d.to(s["x"].dtype)
    u = d if s["scale"] is None else d * s["scale"]
    if s["gate"] is not None:
        t = u * k["a"]
        if case["gate"] == "group":
            t = t.reshape(case["groups"], -1, case["ch"]).sum(dim=1)
        out["dgate"] = (t * _dphi(s["gate"].float(), case["act"])).to(s["gate"].dtype)
        u = u * k["phi"]
    if s["scale"] is not None:
        t = d * k["a"]
        out["dscale"] = (t if s["gate"] is None else t * k["phi"]).sum(dim=0)
    if s["post"] is not None:
        out["dpost_gamma"] = (u * k["yhat"]).sum(dim=0)
        if s["post"][1] is not None:
            out["dpost_beta"] = u.sum(dim=0)
        u = _normalise_back(u * s["post"][0], k["yhat"], k["yr"], kind)
    out["dy"] = u.to(s["y"].dtype)
    return out


def _plain_adam(s):
    g = s["grads"][0]
    norm = _plain_norm(s["grads"])
    g = g * _plain_factor(norm, s["max_norm"])
    s["step"] += 1
    rate = _LR * math.sqrt(1.0 - _BETA2 ** s["step"]) / (1.0 - _BETA1 ** s["step"])
    s["m"].mul_(_BETA1).add_(g, alpha=1.0 - _BETA1)
    s["v"].mul_(_BETA2).add_(g * g, alpha=1.0 - _BETA2)
    s["p"].sub_(rate * s["m"] / (s["v"].sqrt() + _ADAM_EPS))
    s["p_bf16"].copy_(s["p"])
    return norm.float().reshape(1)


def _run_plain(s):
    op = s["case"]["op"]
    if op == "norm":
        return {"norm": _plain_norm(s["grads"]).float().reshape(1)}
    if op == "clip":
        norm = _plain_norm(s["grads"])
        factor = _plain_factor(norm, s["max_norm"])
        out = [(g.float() * factor).to(g.dtype) for g in s["grads"]]
        return {"norm": norm.float().reshape(1), "out": out}
    if op == "adam":
        norm = _plain_adam(s)
        return {"norm": norm, "p": s["p"], "m": s["m"], "v": s["v"], "p_bf16": s["p_bf16"]}
    h, z, k = _plain_forward(s)
    out = {"h": h, "z": z}
    return out if op == "fwd" else {**out, **_plain_backward(s, k)}


# --------------------------------------------------------------------------- the framework's calls
def _run_own(s):
    from pose_estimation_amd import nn, ops

    case = s["case"]
    op = case["op"]
    if op == "norm":
        return {"norm": ops.grad_norm(s["set"])}
    if op == "clip":
        return {"norm": ops.clip_grads(s["set"], s["max_norm"]), "out": s["out"]}
    if op == "adam":
        s["step"] += 1
        norm = ops.adam_step(s["p"], s["m"], s["v"], s["grads"][0], s["step"], _LR, _BETA1, _BETA2,
                             _ADAM_EPS, p_bf16=s["p_bf16"], max_norm=s["max_norm"])
        return {"norm": norm, "p": s["p"], "m": s["m"], "v": s["v"], "p_bf16": s["p_bf16"]}
    kw = dict(norm=case["norm"], post=s["post"], pre=s["pre"], scale=s["scale"], gate=s["gate"],
              gate_act=case["act"])
    h, z, stats = nn.residual_norm(s["y"], s["x"], eps=_EPS, want_stats=op == "train", **kw)
    out = {"h": h, "z": z}
    if op == "train":
        g = nn.residual_norm_bwd(s["dh"], s["dz"], s["y"], s["x"], stats, **kw)
        out.update((k, v) for k, v in g.items() if v is not None)
    return out


def run(state):
    return _run_own(state) if own else _run_plain(state)


# --------------------------------------------------------------------------- 64 bits
def _exact_norm(v, kind, gb):
    centred = v - v.mean(1, True) if kind == "layer" else v
    t = centred / (centred.pow(2).mean(1, True) + _EPS).sqrt() * gb[0]
    return t + gb[1] if gb[1] is not None else t


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("norm", "clip", "adam"):
        wide = [g.double() for g in s["grads"]]
        norm = sum(float((g * g).sum()) for g in wide) ** 0.5
        f = min(1.0, s["max_norm"] / norm)
        told = {"norm": torch.tensor([norm], dtype=torch.float64)}
        if op == "clip":
            told["out"] = [g * f for g in wide]
        if op == "adam":
            t = s["step"] + 1
            m = _BETA1 * s["m"].double() + (1 - _BETA1) * wide[0] * f
            v = _BETA2 * s["v"].double() + (1 - _BETA2) * (wide[0] * f) ** 2
            p = s["p"].double() - _LR * (1 - _BETA2 ** t) ** 0.5 / (1 - _BETA1 ** t) * m / (
                v ** 0.5 + _ADAM_EPS)
            told.update(m=m, v=v, p=p, p_bf16=p)
        return told
    # the definition in float64, its gradients by automatic differentiation
    leaf = {}

    def wide(name, t):
        if t is None:
            return None
        leaf[name] = t.double().requires_grad_(op == "train")
        return leaf[name]

    y, x = wide("dy", s["y"]), wide("dx", s["x"])
    scale, gate = wide("dscale", s["scale"]), wide("dgate", s["gate"])
    post, pre = ([wide("d%s_%s" % (part, n), t) for n, t in zip(("gamma", "beta"), s[part])]
                 if s[part] is not None else None for part in ("post", "pre"))
    branch = y if post is None else _exact_norm(y, case["norm"], post)
    if scale is not None:
        branch = branch * scale
    if gate is not None:
        act = {"none": lambda t: t, "sigmoid": torch.sigmoid, "silu": lambda t: t * torch.sigmoid(t)}
        phi = act[case["act"]](gate)
        if case["gate"] == "group":
            phi = phi[torch.arange(case["rows"], device="cuda") // (case["rows"] // case["groups"])]
        branch = branch * phi
    h = x + branch
    z = None if pre is None else _exact_norm(h, case["norm"], pre)
    told = {"h": h.detach(), "z": None if z is None else z.detach()}
    if op == "train":
        value = (h * s["dh"].double()).sum()
        if z is not None:
            value = value + (z * s["dz"].double()).sum()
        value.backward()
        told.update({k: t.grad for k, t in leaf.items()})
    return told


# --------------------------------------------------------------------------- work
def work(case):
    if case["op"] in ("norm", "clip", "adam"):
        if case["op"] == "adam":
            return {"bytes": 30 * case["total"] + 4, "flops": 16 * case["total"]}
        lengths = _lengths(case["count"], case["total"], case["count"] + case["total"])
        size = sum(n * _BYTES[t] for n, t in zip(lengths, _gradient_types(case)))
        if case["op"] == "norm":
            return {"bytes": size + 4, "flops": 2 * case["total"]}
        return {"bytes": 2 * size + 4, "flops": 3 * case["total"]}
    rows, ch, yb, xb = case["rows"], case["ch"], _BYTES[case["y"]], _BYTES[case["x"]]
    n = rows * ch
    vectors = (int(case["post"]) + int(case["pre"])) * (1 + int(case["bias"])) + int(case["scale"])
    gate = {"none": 0, "row": n, "group": case["groups"] * ch}[case["gate"]] * yb
    pre = int(case["pre"])
    size = n * (yb + 2 * xb + pre * yb) + gate + 4 * ch * vectors
    flops = 20 * n
    if case["op"] == "train":
        size += n * (xb + pre * yb + yb + xb) + gate + 4 * ch * vectors
        flops += 40 * n
    return {"bytes": size, "flops": flops}
