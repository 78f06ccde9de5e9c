"""What the trained-block operators refuse, checked where it needs no GPU: every check stands in front of the first launch."""
import ctypes as C

import pytest
import torch


def _N():
    from diffusion_model_nemo_amd import _native
    return _native


X = 1 << 20   # an address that no call below may reach


def test_layer_norm_entry_points_check_their_arguments():
    lib = _N().lib()
    fwd = lambda x=X, ld=64, y=X, rows=4, width=64, dt=0, at=0: lib.dmn_layer_norm_forward(  # noqa: E731
        x, ld, None, None, y, None, rows, width, dt, at, 1e-5, None)
    assert fwd(x=None) == -1 and fwd(y=None) == -1
    assert fwd(rows=-1) == -1 and fwd(width=0) == -1 and fwd(dt=3) == -1 and fwd(dt=0, at=1) == -1 and fwd(dt=1, at=2) == -1
    assert fwd(ld=63) == -1 and b"row stride" in lib.dmn_last_error()
    assert fwd(rows=1 << 40) == -5
    assert fwd(rows=0, x=None, y=None) == 0                      # nothing to do
    n = lib.dmn_layer_norm_workspace_bytes(1000, 64, 0)
    assert n > 0 and lib.dmn_layer_norm_workspace_bytes(-1, 64, 0) == 0
    bwd = lambda dy=X, stats=X, dw=X, ws=X, nb=n, rows=1000: lib.dmn_layer_norm_backward(  # noqa: E731
        dy, 64, X, 64, None, stats, X, dw, None, rows, 64, 0, 0, ws, nb, None)
    assert bwd(dy=None) == -1 and bwd(stats=None) == -1
    assert bwd(ws=None) == -3 and bwd(nb=n - 1) == -3 and bwd(ws=X + 4) == -3
    assert b"needed" in lib.dmn_last_error()


def test_clip_entry_point_checks_its_arguments():
    N = _N()
    lib = N.lib()
    T = N.DmnGradTensor
    assert C.sizeof(T) == 32
    n = lib.dmn_clip_grads_workspace_bytes(2)

    def call(tensors, inf=0, limit=1.0, scale=1.0, norm=X, ws=X, nb=n):
        arr = (T * len(tensors))(*tensors)
        return lib.dmn_clip_grads(C.addressof(arr), len(tensors), inf, limit, scale, norm, ws, nb, None)

    a, b = T(X, X, 100, 0, 0), T(X + 400, X + 400, 100, 0, 0)
    assert call([a, b], norm=None) == -1 and call([a, b], inf=2) == -1
    assert call([a, b], limit=-1.0) == -1 and call([a, b], limit=float("nan")) == -1 and call([a, b], scale=float("inf")) == -1
    assert call([a, b], nb=n - 1) == -3 and call([a, b], ws=None) == -1
    assert call([a, T(None, X, 5, 0, 0)]) == -1 and call([a, T(X + 402, X + 402, 5, 0, 0)]) == -1   # no address, half an element
    assert call([a, T(X + 400, X + 400, -1, 0, 0)]) == -1 and call([T(X, X, 5, 3, 0)]) == -1
    assert call([a, T(X + 400, None, 100, 0, 0)]) == -1                                             # only one has a destination
    for other in (a, T(X + 396, X + 396, 1, 0, 0), T(X + 398, X + 398, 1, 1, 1)):
        assert call([a, other]) == -1 and b"overlaps" in lib.dmn_last_error()
    assert call([T(X, X, 100, 0, 1)]) == -1 and b"overlaps" in lib.dmn_last_error()                 # in place with another type


def test_operators_refuse_host_tensors_and_bad_arguments():
    from diffusion_model_nemo_amd.modules import LayerNorm, layer_norm
    from diffusion_model_nemo_amd.training import clip_grad_norm_
    x = torch.zeros(2, 8)
    with pytest.raises(RuntimeError, match="no CPU"):
        layer_norm(x)
    with pytest.raises(RuntimeError, match="no CPU"):
        LayerNorm(8)(x)
    with pytest.raises(ValueError):
        LayerNorm(7)(x)
    with pytest.raises(ValueError):
        LayerNorm(0)
    p = torch.nn.Parameter(x)
    assert float(clip_grad_norm_([p], 1.0)) == 0.0       # no gradient anywhere, as in torch
    p.grad = torch.ones(2, 8)
    with pytest.raises(RuntimeError, match="no CPU"):
        clip_grad_norm_([p], 1.0)
    for bad in (dict(max_norm=-1.0), dict(max_norm=float("nan")), dict(max_norm=1.0, grad_scale=float("inf"))):
        with pytest.raises(ValueError):
            clip_grad_norm_([p], **bad)
    assert bool((p.grad == 1).all())


def test_layer_norm_module_has_torch_state():
    from diffusion_model_nemo_amd.modules import LayerNorm
    for kw in ({}, {"bias": False}, {"elementwise_affine": False}):
        ours, theirs = LayerNorm(12, **kw), torch.nn.LayerNorm(12, **kw)
        assert {k: v.shape for k, v in ours.state_dict().items()} == {k: v.shape for k, v in theirs.state_dict().items()}
        ours.load_state_dict(theirs.state_dict())


def test_gradient_clipping_hook_takes_the_configured_value(monkeypatch):
    from diffusion_model_nemo_amd import training
    from diffusion_model_nemo_amd.models import DDPM
    seen = []
    monkeypatch.setattr(training, "clip_grad_norm_", lambda params, value: seen.append((len(params), value)) or torch.tensor(3.0))
    cfg = {"image_size": 32, "timesteps": 10, "channels": 3,
           "diffusion_model": {"_target_": "diffusion_model_nemo.modules.Unet", "input_dim": 32, "dim": 32, "use_convnext": False},
           "sampler": {"_target_": "diffusion_model_nemo.modules.GaussianDiffusion", "timesteps": 10, "schedule_name": "linear"},
           "loss": {"_target_": "diffusion_model_nemo.loss.DiffusionLoss", "loss_type": "l2"}}
    m = DDPM(cfg, trainer={"gradient_clip_val": 0.5})
    opt = torch.optim.SGD(m.parameters(), lr=0.1)
    n = len(list(m.parameters()))
    assert float(m.configure_gradient_clipping(opt)) == 3.0
    m.configure_gradient_clipping(opt, gradient_clip_val=2.0, gradient_clip_algorithm="norm")
    assert seen == [(n, 0.5), (n, 2.0)]
    assert DDPM(cfg).configure_gradient_clipping(opt) is None and len(seen) == 2   # no trainer section: no clipping
    with pytest.raises(NotImplementedError):
        m.configure_gradient_clipping(opt, gradient_clip_algorithm="value")
