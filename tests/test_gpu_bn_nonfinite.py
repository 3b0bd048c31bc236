"""Running batch-norm statistics when a batch is not finite: a channel whose batch mean or variance
is NaN or infinite leaves its running pair as it was, in every form of the finalize, so a training
step that is skipped does not spoil inference and checkpoints for good."""
import math

import pytest
import torch

import pose_estimation_amd as pe
from pose_estimation_amd import nn as pnn

pytestmark = pytest.mark.gpu

C, BAD = 64, [3, 5, 7, 11]


def maps():
    """[2,8,6,C] maps, and a copy whose channels BAD hold a NaN, an infinity, values whose squares
    overflow (a finite mean), and alternating ones whose sum is 0."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    z = torch.randn(2, 8, 6, C, generator=gen, device="cuda").bfloat16()
    bad = z.clone()
    bad[1, 2, 3, 3] = math.nan
    bad[0, 7, 5, 5] = -math.inf
    bad[..., 7] = 1e25
    bad[:, ::2, :, 11], bad[:, 1::2, :, 11] = 1e30, -1e30
    return z, bad


@pytest.mark.parametrize("momentum", [0.1, 0.0])
@pytest.mark.parametrize("form", ["stats", "stats_apply", "finalize", "finalize_apply"])
def test_channels_that_are_not_finite_leave_their_running_pair(form, momentum):
    z, bad = maps()
    gen = torch.Generator(device="cuda").manual_seed(4)
    gamma, beta, rm0 = (torch.randn(C, generator=gen, device="cuda") for _ in range(3))
    rv0 = torch.rand(C, generator=gen, device="cuda") + 0.5
    M = z.numel() // C
    ws, sync = pnn.bn_workspace(M, C, "cuda"), pnn.bn_sync("cuda")
    one = torch.eye(C, device="cuda").bfloat16().view(C, 1, 1, C)

    def run(maps):
        rm, rv, rows = rm0.clone(), rv0.clone(), torch.empty(4, C, device="cuda")
        if form.startswith("finalize"):      # the sums of a conv's epilogue
            w = one
            if maps is bad:                  # 0 * infinity: spoil the filters of BAD instead
                w, maps = one.clone(), z
                for c, v in zip(BAD, (math.nan, math.inf, 1e25, -1e30)):
                    w[c] = v
            maps, n = pnn.conv2d_bnstats(maps, w, ws)
        kw = (gamma, beta, 1e-5, momentum, rm, rv)
        if form == "stats":
            pnn.bn_stats(maps, *kw, ws, out=rows)
        elif form == "stats_apply":
            pnn.bn_stats_apply(maps, *kw, ws, rows, sync)
        elif form == "finalize":
            pnn.bn_finalize(ws, n, M, C, *kw, out=rows)
        else:
            pnn.bn_finalize_apply(ws, n, maps, *kw, rows, sync)
        return rm, rv, rows

    good = torch.tensor([c not in BAD for c in range(C)], device="cuda")
    want, got = run(z), run(bad)
    for a, b, start in zip(got[:2], want[:2], (rm0, rv0)):
        assert torch.equal(a[good], b[good])
        assert torch.equal(a[~good], start[~good])
    assert torch.equal(got[2][:, good], want[2][:, good])
    if momentum:
        assert not bool((want[0] == rm0).any())
    else:
        assert torch.equal(got[0], rm0) and torch.equal(got[1], rv0)


@pytest.mark.parametrize("family,fused", [("resnet50", "0"), ("resnet50", "1"), ("hrnet_w32", "0"),
                                          ("hrnet_w32", "1"), ("mobilenet_v2", "0"),
                                          ("mobilenet_v2", "1")])
def test_a_skipped_step_leaves_a_network_that_predicts_and_trains(family, fused, monkeypatch):
    monkeypatch.setenv("PE_BN_FUSED", fused)
    model = {"layers": [1, 1, 1, 1], "head_channels": 64} if family == "resnet50" else {
        "backbone": family, "width": 32, "modules": [1, 1, 1], "blocks": 1, "layer1_blocks": 1}
    t = pe.Trainer({"train_config": {"batch_size": 2, "skip_nonfinite_steps": True,
                                     "preprocess": {"image_resize": [64, 64]}},
                    "model_config": model})
    t.build_model(seed=3)
    net = t.net
    features, labels = next(t.get_features_labels_data(1))
    t.train_step(features, labels)
    assert math.isfinite(float(t.grad_norm))

    def state():
        return {"master": net.master, "opt_m": net.opt_m, "opt_v": net.opt_v,
                **{"mean." + k: v for k, v in net.bn_mean.items()},
                **{"var." + k: v for k, v in net.bn_var.items()}}

    keep = {k: v.clone() for k, v in state().items()}
    net.work.fill_(math.nan)                 # as if every activation had overflowed
    t.train_step(features, labels)
    assert not math.isfinite(float(t.grad_norm))
    for k, v in state().items():
        assert torch.equal(v, keep[k]), k
    net.work.copy_(net.master)
    net.refresh_transposes()
    t.train_step(features, labels)
    assert math.isfinite(float(t.grad_norm))
    assert not torch.equal(net.master, keep["master"])
    for k, v in state().items():
        assert bool(v.isfinite().all()), k
    assert bool(t.predict(features["images"]).isfinite().all())
