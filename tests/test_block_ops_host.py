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


def test_linear_entry_points_check_their_arguments():
    lib = _N().lib()
    need = lib.dmn_linear_forward_workspace_bytes
    assert need(X, 1024, X, 64, 1024, 1024, 1) == 0                   # few rows: no workspace
    assert need(X, 4096, X, 256, 4096, 256, 1) > 0                    # k is split
    assert need(X, 1000, X, 4096, 1000, 4096, 1) == 0                 # rows of whole 16-byte pieces
    odd = need(X, 1001, X, 4096, 1001, 4096, 1)
    assert odd >= (4096 + 4096) * 1008 * 2 and need(X + 2, 1000, X, 4096, 1000, 4096, 1) >= 4096 * 1000 * 2
    for bad in ((X, 8, X, -1, 8, 8, 0), (X, 8, X, 100, 0, 8, 0), (X, 8, X, 100, 8, 8, 3), (X, 8, X, 1 << 27, 8, 8, 0)):
        assert need(*bad) == 0
    fwd = lambda x=X, ldx=1001, w=X, res=None, ldr=0, y=X, rows=4096, k=1001, n=4096, act=0, dt=1, ws=X, nb=odd: lib.dmn_linear_forward(  # noqa: E731
        x, ldx, w, None, res, ldr, y, None, rows, k, n, act, dt, ws, nb, None)
    assert fwd(x=None) == -1 and fwd(w=None) == -1 and fwd(y=None) == -1
    assert fwd(act=4) == -1 and fwd(act=-1) == -1 and fwd(dt=3) == -1 and fwd(rows=-1) == -1 and fwd(k=0) == -1 and fwd(n=0) == -1
    assert fwd(ldx=1000) == -1 and fwd(res=X, ldr=4095) == -1
    assert fwd(ldx=1 << 20) == -5 and fwd(rows=1 << 27) == -5 and fwd(k=1 << 20, ldx=1 << 20) == -5
    assert fwd(ws=None) == -3 and fwd(nb=odd - 1) == -3 and fwd(ws=X + 16) == -3 and b"needed" in lib.dmn_last_error()
    assert fwd(rows=0, x=None, w=None, y=None) == 0
    n = lib.dmn_linear_backward_workspace_bytes(X, 4096, X, 1001, X, 4096, 1001, 4096, 3, 1)
    bwd = lambda dy=X, lddy=4096, x=X, w=X, z=X, dx=X, dw=X, db=X, rows=4096, act=3, ws=X, nb=n: lib.dmn_linear_backward(  # noqa: E731
        dy, lddy, x, 1001, w, z, dx, dw, db, rows, 1001, 4096, act, 1, ws, nb, None)
    assert bwd(dy=None) == -1 and bwd(x=None) == -1 and bwd(w=None) == -1 and bwd(z=None) == -1 and bwd(act=5) == -1
    assert bwd(lddy=4095) == -1 and bwd(lddy=1 << 20) == -5
    assert bwd(ws=None) == -3 and bwd(nb=n - 1) == -3 and bwd(ws=X + 128) == -3
    assert bwd(dx=None, dw=None, db=None, dy=None) == 0


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


def test_linear_refuses_host_tensors_and_unknown_activations():
    from diffusion_model_nemo_amd.modules import Linear, linear
    with pytest.raises(RuntimeError, match="no CPU"):
        linear(torch.zeros(2, 8), torch.zeros(4, 8))
    with pytest.raises(RuntimeError, match="no CPU"):
        Linear(8, 4)(torch.zeros(2, 8))
    with pytest.raises(ValueError):
        Linear(8, 4, activation="tanh")
    ours, theirs = Linear(8, 4, bias=False, activation="gelu"), torch.nn.Linear(8, 4, bias=False)
    ours.load_state_dict(theirs.state_dict())


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


def test_linear_entry_points_take_the_exact_flag():
    lib = _N().lib()
    need = lambda act, dt: lib.dmn_linear_backward_workspace_bytes(X, 4096, X, 1024, X, 4096, 1024, 4096, act, dt)  # noqa: E731
    dz = 4096 * 4096 * 2
    assert need(3 + 16, 1) - need(3, 1) >= dz and need(3 + 16, 2) - need(3, 2) >= dz     # dz in two parts, or one
    assert need(0, 1) == need(16, 1) and need(3, 0) == need(3 + 16, 0)
    for act in (20, 31, 32, 8, -16):
        assert lib.dmn_linear_backward(X, 8, X, 8, X, X, X, X, X, 4, 8, 8, act, 1, None, 0, None) == -1
        assert lib.dmn_linear_forward(X, 8, X, None, None, 0, X, None, 4, 8, 8, act, 1, None, 0, None) == -1


def test_default_stream_is_never_recorded():
    assert _N().lib().dmn_stream_is_capturing(None) == 0


def _unrecorded_calls(device):
    """name -> (the call on one tensor, that tensor): every input of layer_norm and linear in turn."""
    ops = _N().ops()
    x, w, v, r = (torch.ones(s, device=device) for s in ((4, 8), (8, 8), (8,), (4, 8)))
    s = 0 if device == "cpu" else torch._C._cuda_getCurrentRawStream(0)
    return {"layer_norm x": (lambda t: ops.layer_norm(t, v, v, 1e-5, s), x), "layer_norm weight": (lambda t: ops.layer_norm(x, t, None, 1e-5, s), v),
            "layer_norm bias": (lambda t: ops.layer_norm(x, None, t, 1e-5, s), v), "linear x": (lambda t: ops.linear(t, w, v, 3, r, s), x),
            "linear weight": (lambda t: ops.linear(x, t, None, 0, None, s), w), "linear bias": (lambda t: ops.linear(x, w, t, 1, None, s), v),
            "linear residual": (lambda t: ops.linear(x, w, None, 0, t, s), r)}


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_forward_mode_derivatives_and_traces_are_refused(device):
    """They would come out as a derivative of zero, and as a traced module that returns memory nobody wrote."""
    from torch.autograd import forward_ad
    from diffusion_model_nemo_amd.training import clip_grad_norm_
    for name, (call, t) in _unrecorded_calls(device).items():
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(t, torch.ones_like(t))
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(dual)
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(call, (t,), check_trace=False)
    p = torch.nn.Parameter(torch.ones(4, device=device))
    p.grad = torch.ones(4, device=device)
    for finite in (False, True):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(lambda t: t + clip_grad_norm_([p], 1.0, error_if_nonfinite=finite), (p.detach(),), check_trace=False)
    assert bool((p.grad == 1).all())


def test_gradient_clipping_hook_works_beside_any_optimizer(monkeypatch):
    """The hook is the autograd route's, with whatever torch optimizer and learning-rate policy the config names."""
    from diffusion_model_nemo_amd import training
    from diffusion_model_nemo_amd.models import DDPM
    seen = []
    monkeypatch.setattr(training, "clip_grad_norm_", lambda params, value: seen.append(value) or torch.tensor(3.0))
    cfg = {"image_size": 32, "timesteps": 10, "channels": 3, "optim": {"name": "sgd", "lr": 0.1, "sched": {"name": "StepLR"}},
           "diffusion_model": {"_target_": "diffusion_model_nemo.modules.Unet", "input_dim": 32, "dim": 32, "use_convnext": False},
           "sampler": {"_target_": "diffusion_model_nemo.modules.GaussianDiffusion", "timesteps": 10, "schedule_name": "linear"},
           "loss": {"_target_": "diffusion_model_nemo.loss.DiffusionLoss", "loss_type": "l2"}}
    m = DDPM(cfg, trainer={"gradient_clip_val": 0.5})
    assert float(m.configure_gradient_clipping(torch.optim.SGD(m.parameters(), lr=0.1))) == 3.0 and seen == [0.5]
    assert DDPM(cfg).configure_gradient_clipping(torch.optim.SGD(m.parameters(), lr=0.1)) is None
    with pytest.raises(NotImplementedError):
        m._optim_settings()          # the all-device step stays AdamW


def test_configured_clipping_by_value_is_refused_instead_of_clipped_by_norm(monkeypatch):
    from diffusion_model_nemo_amd import training
    from diffusion_model_nemo_amd.models import DDPM
    seen = []
    monkeypatch.setattr(training, "clip_grad_norm_", lambda params, value: seen.append(value) or torch.tensor(3.0))
    cfg = {"image_size": 32, "timesteps": 10, "channels": 3,
           "diffusion_model": {"_target_": "diffusion_model_nemo.modules.Unet", "input_dim": 32, "dim": 32, "use_convnext": False},
           "sampler": {"_target_": "diffusion_model_nemo.modules.GaussianDiffusion", "timesteps": 10, "schedule_name": "linear"},
           "loss": {"_target_": "diffusion_model_nemo.loss.DiffusionLoss", "loss_type": "l2"}}
    m = DDPM(cfg, trainer={"gradient_clip_val": 0.5, "gradient_clip_algorithm": "value"})
    opt = torch.optim.SGD(m.parameters(), lr=0.1)
    for kw in ({}, {"gradient_clip_val": 2.0}):
        with pytest.raises(NotImplementedError, match="value"):
            m.configure_gradient_clipping(opt, **kw)
    with pytest.raises(NotImplementedError, match="value"):
        m._optim_settings()
    assert m.configure_gradient_clipping(opt, gradient_clip_val=0.0) is None and not seen
    m.configure_gradient_clipping(opt, gradient_clip_algorithm="norm")       # the caller's word is the last
    assert seen == [0.5]
    assert DDPM(cfg, trainer={"gradient_clip_algorithm": "value"}).configure_gradient_clipping(opt) is None


def test_m0_belongs_to_the_requests_that_write_it():
    """Their inline assembly overwrites m0 and cannot declare it: nothing else in those kernels may use it."""
    from diffusion_model_nemo_amd import isa_check
    assert isa_check.assert_m0_is_the_requests_own(_N().LIB_PATH) >= 40
    own = ["s_mov_b32 m0, s4", "s_nop 4", "buffer_load_dwordx4 v3, s[8:11], 0 offen lds"]
    kernel = lambda *code: "0000000000001000 <_ZN1a16gemm_pipe_kernelIfEEv>:\n" + "".join(f"\t{c} // 000000001000: BF800004\n" for c in code)  # noqa: E731
    bad = lambda *code: list(isa_check.foreign_m0_uses(kernel(*code)).values())  # noqa: E731
    assert bad("v_add_f32_e32 v0, v1, v2", *own, *own) == [[]]
    assert bad(*own, "s_mov_b32 s3, m0") == [["s_mov_b32 s3, m0"]]                     # somebody keeps a value there
    assert bad("s_mov_b32 m0, -1", *own) == [["s_mov_b32 m0, -1"]]
    assert bad(own[0], "s_nop 0", own[2]) == [[own[0]]] and bad(own[0], own[1]) == [[own[0]]]
    assert isa_check.foreign_m0_uses(kernel(*own).replace("gemm_pipe", "other")) == {}


def test_every_compiled_tile_has_a_tested_size():
    """The sizes of test_every_tile_type_and_layout against the planner: a change of its model must not move them off a kernel."""
    from test_gpu_block_mends import EVERY_TILE
    lib = _N().lib()
    seen = set()
    for m, k, n, kind in EVERY_TILE:
        act = 0 if kind is None else 3 + 16
        for dt in range(3) if act == 0 else (1, 2):
            for alone in (0, 1):
                p = (C.c_int * 7)()
                assert lib.dmn_test_linear_plan(m, k, n, act, dt, alone, p) == 0
                two = act > 0
                seen.add(("forward", dt, p[0]))
                seen.add(("forward split", dt, p[0] if p[1] > 1 else None))
                if p[2]:
                    seen |= {("pair", dt, two, p[3]), ("pair split", dt, two, p[3], p[4] > 1, p[6] > 1)}
                else:
                    seen |= {("dx", dt, two, p[3]), ("dw", dt, two, p[5]), ("dx split", dt, two, p[3], p[4] > 1), ("dw split", dt, two, p[5], p[6] > 1)}
                    if not alone:
                        seen.add(("one after the other", dt, two))
    for dt in range(3):
        want = {("forward", dt, t) for t in (-1, 0, 1, 2, 3)} | {("forward split", dt, t) for t in (0, 1, 2, 3)}
        for two in (False, True)[:1 if dt == 0 else 2]:
            want |= {(op, dt, two, t) for op in ("dx", "dw") for t in range(4)} | {("pair", dt, two, t) for t in (2, 3)} | {("one after the other", dt, two)}
            want |= {(op + " split", dt, two, t, True) for op in ("dx", "dw") for t in range(4) if not (op == "dw" and t == 2 and not two and dt)}
            want |= {("pair split", dt, two, t, a, b) for t in (2, 3) for a in (False, True) for b in (False, True)}
        assert want <= seen, sorted(map(str, want - seen))
    p = (C.c_int * 7)()
    assert lib.dmn_test_linear_plan(0, 8, 8, 0, 0, 0, p) == -1 and lib.dmn_test_linear_plan(8, 8, 8, 4, 0, 0, p) == -1
    assert lib.dmn_test_linear_plan(8, 8, 8, 0, 0, 0, None) == -1
