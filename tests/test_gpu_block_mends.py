"""Calls of the trained-block operators at the edges of their types, tiles and autograd modes, against the formulas in float64
with the bounds of `check_linear` (tests/test_gpu_block_ops.py), or as refusals."""
import pytest
import torch

from test_gpu_block_ops import BF, F32, HF, TYPES, U, act_formula, close, floor_of, half_step, product, randn

pytestmark = pytest.mark.gpu


def grads_of(x, w, b, kind, dy, **kw):
    from diffusion_model_nemo_amd.modules import linear
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    y = linear(*leaves, kind, **kw)
    return (y.detach(),) + torch.autograd.grad(y, leaves, dy)


@pytest.mark.parametrize("rows", [5, 80], ids=["few", "tiles"])
@pytest.mark.parametrize("kind", ["relu", "silu", "gelu"])
def test_float16_sums_beyond_its_range_have_finite_gradients(kind, rows):
    """Column 0 sums to -72000, column 1 to 72000 (float16 ends at 65504), the others stay small. The slopes there are 0 and 1,
    so column 0 adds nothing to any gradient and column 1 adds dy."""
    x, w = torch.zeros((rows, 24), dtype=HF, device="cuda"), randn((40, 24), 1, HF, 0.1)
    x[:, 1:] = randn((rows, 23), 2, HF)
    x[:, 0], w[:, 0] = 240.0, 0.0
    w[0], w[1] = 0.0, 0.0
    w[0, 0], w[1, 0] = -300.0, 300.0
    b, dy = randn((40,), 3, HF), randn((rows, 40), 4, HF)
    y, dx, dw, db = grads_of(x, w, b, kind, dy)
    z = product(x, w.t())[0] + b.double()
    a, slope = act_formula(z, kind)
    want = dy.double() * slope
    assert float(z[:, 0].max()) < -65520 and float(z[:, 1].min()) > 65520
    assert not bool(y[:, 0].any()) and bool(torch.isinf(y[:, 1]).all())
    # per element of dz: half a step of z (at most 5 here) through a slope that changes by at most 1.2, the activation's own
    # 1e-5 and dz's rounding; one rounding of the result, and of the float32 sums much less
    edz = dy.double().abs() * (1.2 * half_step(HF) * 5 + 1e-5) + half_step(HF) * want.abs() + floor_of(HF)
    edz[:, :2] = half_step(HF) * want[:, :2].abs() + floor_of(HF)
    if kind == "relu":
        edz = torch.where(z.abs() <= 1e-4, dy.double().abs(), edz)
    for got, full, err, size in ((dx, product(want, w)[0], edz @ w.double().abs(), product(want, w)[1]),
                                 (dw, product(want.t(), x)[0], edz.t().contiguous() @ x.double().abs(), product(want.t(), x)[1]),
                                 (db, want.sum(0), edz.sum(0), want.abs().sum(0))):
        close(got, full, half_step(HF) * full.abs() + err + 200 * U * size + floor_of(HF), kind)
    assert not bool(dw[0].any()) and not bool(db[0].any())


@pytest.mark.parametrize("kind", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_slopes_at_infinite_sums_are_their_limits(dtype, kind):
    x = torch.ones((70, 8), dtype=dtype, device="cuda")
    w = torch.zeros((12, 8), dtype=dtype, device="cuda")
    b = torch.zeros((12,), dtype=dtype, device="cuda")
    b[3], b[4], b[5] = float("inf"), float("-inf"), float("nan")
    dy = torch.ones((70, 12), dtype=dtype, device="cuda")
    db = grads_of(x, w, b, kind, dy)[3]
    assert float(db[3]) == 70 and float(db[4]) == 0 and bool(torch.isnan(db[5]))
    assert bool((db[6:] == 35).all()) and bool((db[:3] == 35).all())


# rows, in, out, activation: together they take every compiled tile in every type and operand layout, with k whole and split, dx and
# dweight in one launch, one after the other and alone, dz in one part and in two (test_block_ops_host.py asserts it).
EVERY_TILE = [(1, 33, 33, None), (1, 33, 33, "gelu"), (1, 33, 520, "gelu"), (1, 33, 1016, None), (510, 33, 33, "gelu"), (1020, 33, 33, None),
              (20, 4104, 33, None), (1, 1016, 16360, "gelu"), (1, 1016, 4104, None), (1, 1016, 4104, "gelu"), (1, 2040, 16360, None),
              (1020, 33, 520, "gelu"), (321, 136, 16360, "gelu"), (1020, 16360, 250, None), (4090, 1016, 1016, "gelu"), (321, 16360, 136, "gelu"),
              (8184, 250, 8184, None), (2050, 2040, 33, None), (4090, 33, 2040, None), (8184, 136, 8184, "gelu"), (1020, 16360, 1016, "gelu"),
              (1030, 2040, 2040, None), (8184, 520, 8184, None), (130, 16360, 8184, "gelu"), (8184, 16360, 136, "gelu"), (250, 1016, 16360, None),
              (8184, 1016, 16360, None), (8184, 16360, 1016, None), (16368, 504, 16360, None), (321, 8184, 1016, "gelu"),
              (8184, 136, 8184, None), (120, 8184, 16360, None), (4090, 1016, 1016, None)]


def check_gradients(m, k, n, dtype, kind, rounded=False, scale=1.0, one_by_one=False):
    """dx, dweight and dbias with ONE rounding (the result's) and float32 work in front of it; `rounded` adds half a step of z and
    of dz. Two numbers of the type hold dz to half_step squared of it (float16: down to 2^-35, as its low part is kept 2^11
    times larger and both are halved)."""
    from diffusion_model_nemo_amd.modules import linear
    x, w, b = randn((m, k), 1, dtype), randn((n, k), 2, dtype, k ** -0.5), randn((n,), 3, dtype, 0.3)
    dy = randn((m, n), 4, dtype, scale)
    got = grads_of(x, w, b, kind, dy, rounded_backward=rounded)
    alone = ()
    if one_by_one:   # each product in a launch of its own too
        for i in range(2):
            leaves = [t.detach().requires_grad_(i == j) for j, t in enumerate((x, w, b))]
            alone += torch.autograd.grad(linear(*leaves, kind, rounded_backward=rounded), leaves[i], dy)
    z, za = product(x, w.t())
    ez = (k + 64) * U * za + 4 * U * (z.abs() + 2 * b.double().abs())
    z = z + b.double()
    a, slope = act_formula(z, kind)
    close(got[0], a, half_step(dtype) * a.abs() + 1.13 * ez + 6e-6 * a.abs() + floor_of(dtype), "y")
    d = dy.double()
    dz, h = d * slope, half_step(dtype)
    edz = d.abs() * (1.2 * ez + 4e-6 + 4 * U)
    if rounded:
        edz = edz + d.abs() * 1.2 * (h * z.abs() + floor_of(dtype))
    if kind == "relu":   # the slope jumps at 0: only where the sign is in doubt, and there by all of dy
        edz = torch.where(z.abs() <= ez + (floor_of(dtype) if rounded else 0), d.abs(), torch.zeros_like(dz))
    if kind is None:     # dz is dy itself
        edz = torch.zeros_like(dz)
    part = edz if kind is None else h * dz.abs() + floor_of(dtype) if rounded else h * h * dz.abs() + (2.0 ** -35 if dtype == HF else 2.0 ** -140)
    for at, (p, q), depth in ((1, (dz, w), n), (2, (dz.t(), x), m)):
        want, size = product(p, q)
        err = product((edz + part) if at == 1 else (edz + part).t(), q)[1]
        tol = h * want.abs() + err + (2 * depth + 64) * U * (1.01 * size + err) + floor_of(dtype)
        once = (want.to(dtype).double() - want).norm()
        for g in (got[at],) + alone[at - 1:at]:
            close(g, want, tol, "dx" if at == 1 else "dw")
            if not rounded and kind != "relu" and scale == 1.0 and dtype != F32:
                # all errors together, against those of the exact result rounded once
                assert float((g.double() - want).norm()) <= 1.02 * float(once), at
    want = dz.sum(0)
    close(got[3], want, h * want.abs() + edz.sum(0) + (m + 64) * U * (dz.abs() + edz).sum(0) + floor_of(dtype), "db")


@pytest.mark.parametrize("dtype", [BF, HF], ids=str)
@pytest.mark.parametrize("kind", ["silu", "gelu"])
@pytest.mark.parametrize("m,k,n", [(1, 8, 8), (17, 40, 24), (130, 127, 131), (70, 96, 104), (2048, 512, 1024), (64, 72, 8200), (8200, 72, 64)])
def test_gradients_of_16_bit_layers_are_rounded_once(dtype, kind, m, k, n):
    check_gradients(m, k, n, dtype, kind)


@pytest.mark.parametrize("dtype", [BF, HF], ids=str)
@pytest.mark.parametrize("m,k,n", [(130, 127, 131), (64, 72, 8200), (8200, 72, 64), (1030, 1032, 1040)])
def test_gradients_of_16_bit_layers_one_by_one(dtype, m, k, n):
    check_gradients(m, k, n, dtype, "gelu", one_by_one=True)
    check_gradients(m, k, n, dtype, "relu", one_by_one=True)


@pytest.mark.parametrize("m,k,n,kind", EVERY_TILE)
def test_every_tile_type_and_layout(m, k, n, kind):
    for dtype in TYPES if kind is None else (BF, HF):
        check_gradients(m, k, n, dtype, kind, one_by_one=True)


@pytest.mark.parametrize("m,k,n,kind,tiles", [(4096, 1024, 4096, None, (0, None)), (2048, 2048, 2048, None, (1, None)), (4096, 4096, 4096, None, (0, 0)),
                                              (4096, 4096, 4096, "gelu", (0, 0)), (250, 1016, 16360, None, (1, None))])
def test_large_tiles_are_captured(m, k, n, kind, tiles):
    """Tiles of more LDS than a launch may have without an attribute: set inside a capture, forward and backward."""
    import ctypes as C
    from diffusion_model_nemo_amd import _native as N
    from diffusion_model_nemo_amd.modules import linear
    plan = (C.c_int * 7)()
    assert N.lib().dmn_test_linear_plan(m, k, n, 0 if kind is None else 3 + 16, 1, 0, plan) == 0
    assert plan[0] == tiles[0] and (tiles[1] is None or (plan[2], plan[3]) == (0, tiles[1])), list(plan)
    x, w = randn((m, k), 1, BF).requires_grad_(True), randn((n, k), 2, BF, k ** -0.5).requires_grad_(True)
    dy = randn((m, n), 4, BF)

    def step():
        y = linear(x, w, None, kind)
        return (y.detach(),) + torch.autograd.grad(y, (x, w), dy)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for turn in range(3):
        with torch.no_grad():
            x.copy_(randn((m, k), 20 + turn, BF))
        graph.replay()
        kept = [g.clone() for g in got]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(kept, want)), turn


@pytest.mark.parametrize("scale", [1e-6, 2e-4])
def test_small_float16_gradients_keep_their_digits(scale):
    check_gradients(300, 136, 520, HF, "gelu", scale=scale)


def test_large_float16_gradients_stay_in_range():
    """A slope of up to 1.13 takes dz out of float16's range where dx is well within it."""
    x, w, b = torch.full((80, 8), 0.25, dtype=HF, device="cuda"), torch.full((16, 8), 0.5, dtype=HF, device="cuda"), torch.full((16,), 0.5, dtype=HF, device="cuda")
    w[8:] = -0.5
    dy = torch.full((80, 16), 65000.0, dtype=HF, device="cuda")
    b[8:] = 2.5                                                         # sums of 1.5: gelu's slope is 1.1275 there
    y, dx, dw, db = grads_of(x, w, b, "gelu", dy)
    assert bool((dx == 0).all())                                        # 8 times 0.5 dz - 8 times 0.5 dz


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("kind", ["relu", "gelu"])
def test_rounded_backward_is_the_callers_choice(dtype, kind):
    from diffusion_model_nemo_amd.modules import Linear, linear
    for m, k, n in ((1, 8, 8), (130, 127, 131), (2048, 512, 1024), (64, 72, 8200)):
        check_gradients(m, k, n, dtype, kind, rounded=True)
    layer = Linear(96, 104, activation=kind, dtype=dtype, device="cuda", rounded_backward=True)
    x, dy = randn((70, 96), 1, dtype).requires_grad_(True), randn((70, 104), 2, dtype)
    want = grads_of(x, layer.weight, layer.bias, kind, dy, rounded_backward=True)
    y = layer(x)
    assert torch.equal(y, want[0]) and all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, (x, layer.weight, layer.bias), dy), want[1:]))
    if dtype == TYPES[0]:   # float32: there is nothing to choose
        assert all(torch.equal(p, q) for p, q in zip(grads_of(x, layer.weight, layer.bias, kind, dy), want))
    assert torch.equal(linear(x, layer.weight, layer.bias, None, rounded_backward=True), linear(x, layer.weight, layer.bias))


def test_capture_guard_sees_leaves_behind_views_and_copies():
    """A transposed weight, a view of an input and a strided bias are no leaves themselves; their gradients end in leaves all the same."""
    from diffusion_model_nemo_amd.modules import layer_norm, linear
    x, w, b = randn((130, 72), 1).requires_grad_(True), randn((72, 40), 2, scale=0.1).requires_grad_(True), randn((80,), 3).requires_grad_(True)
    plain, fixed = randn((130, 72), 4), randn((40, 72), 5)
    dy = randn((130, 40), 6)
    calls = {"transposed weight": (lambda: linear(plain, w.t(), None, "gelu"), w), "strided bias": (lambda: linear(plain, fixed, b[::2]), b),
             "view of x": (lambda: linear(x.view(13, 10, 72).reshape(130, 72) * 2, fixed), x),
             "rows of x": (lambda: layer_norm(x[3:]), x), "strided scale": (lambda: layer_norm(randn_40, b[::2]), b)}
    randn_40 = randn((9, 40), 7)
    for name, (call, leaf) in calls.items():
        alive = call()
        with pytest.raises(RuntimeError, match="still lives"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
        del alive
    # with the eager graphs gone: captured, replayed, and as the eager call
    def step():
        y = linear(x * 1.0, w.t(), b[::2], "gelu")
        return (y.detach(),) + torch.autograd.grad(y, (x, w, b), dy)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        got = step()
    for turn in range(3):
        with torch.no_grad():
            x.copy_(randn((130, 72), 20 + turn))
        graph.replay()
        kept = [g.clone() for g in got]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(kept, want)), turn


def test_forward_alone_is_captured_beside_an_eager_graph_and_on_a_forked_stream():
    from diffusion_model_nemo_amd.modules import layer_norm, linear
    x, w = randn((70, 72), 1).requires_grad_(True), randn((40, 72), 2, scale=0.1).requires_grad_(True)
    alive = linear(layer_norm(x), w)
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        y = linear(layer_norm(x), w)
    for turn in range(3):
        with torch.no_grad():
            x.copy_(randn((70, 72), 10 + turn))
        graph.replay()
        kept = y.clone()
        with torch.no_grad():
            assert torch.equal(kept, linear(layer_norm(x), w)), turn
    del alive
    # a leaf whose first use lies on a stream that was forked into the capture itself
    graph, fork = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        fork.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(fork):
            a = linear(x, w)
        torch.cuda.current_stream().wait_stream(fork)
        b = linear(x, w, activation="relu")
        kept = (a.detach(), b.detach())
        del a, b
    graph.replay()
    with torch.no_grad():
        assert torch.equal(kept[0], linear(x, w)) and torch.equal(kept[1], linear(x, w, activation="relu"))


@pytest.mark.parametrize("op", ["linear", "layer_norm"])
def test_captured_backward_of_an_eager_forward(op):
    """Forward made eagerly on a stream, its backward captured there: refused while a leaf it ends in was first used on the default
    stream by a graph that still lives, unless the gradients asked for do not pass that leaf."""
    from diffusion_model_nemo_amd.modules import layer_norm, linear
    x = randn((70, 72), 1).requires_grad_(True)
    w = randn((72, 72), 2, scale=0.1).requires_grad_(True) if op == "linear" else randn((72,), 2).requires_grad_(True)
    dy = randn((70, 72), 3)
    call = (lambda h: linear(h, w)) if op == "linear" else (lambda h: layer_norm(h, w))
    side = torch.cuda.Stream()
    alive = call(x)
    want = torch.autograd.grad(alive, (x, w), dy, retain_graph=True)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = call(x)
    with pytest.raises(RuntimeError, match="still lives"):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
            torch.autograd.grad(y, (x, w), dy, retain_graph=True)
    del y
    with torch.cuda.stream(side):
        h = x.detach().clone().requires_grad_(True)
        y = call(h)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        (dx,) = torch.autograd.grad(y, (h,), dy, retain_graph=True)   # w's gradient is not asked for
    for turn in range(3):
        dx.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(dx, want[0]), turn
    del y, alive
    with torch.cuda.stream(side):
        y = call(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
    for turn in range(3):
        for g in got:
            g.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want)), turn


@pytest.mark.parametrize("kind", [None, "gelu"])
def test_linear_keeps_only_what_its_gradients_need(kind):
    """A frozen layer's input may be overwritten before the backward, and the weight of a layer whose input needs no gradient, as with
    torch's own linear layer; what a gradient does need is still guarded."""
    from diffusion_model_nemo_amd.modules import linear
    x, w, b, r, dy = randn((70, 72), 1), randn((40, 72), 2, scale=0.1), randn((40,), 3), randn((70, 40), 4), randn((70, 40), 5)
    want = torch.autograd.grad(linear(*(t.requires_grad_(True) for t in (x, w, b)), kind, r.requires_grad_(True)), (x, w, b, r), dy)
    for i, harmless in enumerate(((0, 2, 3), (1, 2, 3), (0, 1, 2, 3), (0, 1, 2, 3))):
        args = [t.detach().clone().requires_grad_(i == j) for j, t in enumerate((x, w, b, r))]
        y = linear(args[0], args[1], args[2], kind, args[3])
        with torch.no_grad():
            for j in harmless:
                args[j].add_(1.0)
        (got,) = torch.autograd.grad(y, args[i], dy, retain_graph=True)
        assert torch.equal(got, want[i]), i
        for j in set(range(2)) - set(harmless):
            with torch.no_grad():
                args[j].add_(1.0)
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                torch.autograd.grad(y, args[i], dy, retain_graph=True)
    frozen, given = torch.nn.Parameter(w.detach().clone(), requires_grad=False), x.detach().clone().requires_grad_(True)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = linear(given * 1.0, frozen)
    assert torch.cuda.memory_allocated() - before <= y.numel() * y.element_size() + 512     # the product's input is gone again


def test_c_callers_keep_a_rounded_z_unless_they_ask():
    """z of the operands' type and a rounded dz without DMN_LINEAR_EXACT, as `rounded_backward=True` computes them."""
    from diffusion_model_nemo_amd import _native as N
    lib, s = N.lib(), N.current_stream_handle()
    m, k, n = 130, 72, 88
    x, w, b, dy = randn((m, k), 1, BF), randn((n, k), 2, BF, 0.1), randn((n,), 3, BF), randn((m, n), 4, BF)
    for flag, rounded in ((0, True), (16, False)):
        z = torch.empty((m + 1, n), dtype=BF if rounded else torch.float32, device="cuda")
        z[m] = 7.0
        y, dx, dw, db = (torch.empty_like(t) for t in (dy, x, w, b))
        nb = max(lib.dmn_linear_forward_workspace_bytes(x.data_ptr(), k, w.data_ptr(), m, k, n, 1),
                 lib.dmn_linear_backward_workspace_bytes(dy.data_ptr(), n, x.data_ptr(), k, w.data_ptr(), m, k, n, 3 + flag, 1))
        ws = torch.empty(nb, dtype=torch.uint8, device="cuda")
        N.check(lib.dmn_linear_forward(x.data_ptr(), k, w.data_ptr(), b.data_ptr(), None, 0, y.data_ptr(), z.data_ptr(), m, k, n, 3 + flag, 1,
                                       ws.data_ptr(), nb, s))
        N.check(lib.dmn_linear_backward(dy.data_ptr(), n, x.data_ptr(), k, w.data_ptr(), z.data_ptr(), dx.data_ptr(), dw.data_ptr(), db.data_ptr(),
                                        m, k, n, 3 + flag, 1, ws.data_ptr(), nb, s))
        want = grads_of(x, w, b, "gelu", dy, rounded_backward=rounded)
        assert all(torch.equal(p, q) for p, q in zip((y, dx, dw, db), want)) and bool((z[m] == 7.0).all())


@pytest.mark.parametrize("width", [1, 24])
def test_views_with_the_negation_bit_are_read_with_their_sign(width):
    """What torch.conj(z).imag gives: memory that holds the negative of the values."""
    from diffusion_model_nemo_amd.modules import layer_norm, linear
    from diffusion_model_nemo_amd.training import clip_grad_norm_
    x, w, b, r, dy = randn((9, width), 1), randn((width, width), 2), randn((width,), 3), randn((9, width), 4), randn((9, width), 5)
    neg = [torch._neg_view(t) for t in (x, w, b, r, dy)]
    for t in neg:
        assert t.is_neg() and t.is_contiguous()
    plain = [t.clone() for t in neg]
    assert torch.equal(plain[0], -x) and not plain[0].is_neg()
    strided = torch.complex(x, r).conj().imag                       # rows two elements apart
    assert strided.is_neg() and torch.equal(linear(strided, w), linear(-r, w)) and torch.equal(layer_norm(strided), layer_norm(-r))

    def both(op, n):
        out = []
        for args in (neg, plain):
            leaves = [t.detach().requires_grad_(True) for t in args[:n]]
            y = op(*leaves)
            out.append((y,) + torch.autograd.grad(y, leaves, args[4]))
        assert all(torch.equal(p, q) for p, q in zip(*out))

    both(lambda x, w, b, r: linear(x, w, b, "gelu", r), 4)
    both(lambda x, w, b: layer_norm(x, w[0], b), 3)
    p = [torch.nn.Parameter(torch.zeros_like(t)) for t in (x, r)]
    p[0].grad, p[1].grad = neg[0], r.clone()
    norm = clip_grad_norm_(p, 0.5)
    want = torch.linalg.vector_norm(torch.cat([plain[0], r]).double())
    assert abs(float(norm) - float(want)) <= 4 * U * float(want)
    close(p[0].grad.clone(), plain[0].double() * 0.5 / want, 8 * U * plain[0].double().abs(), "clipped")
    out = [torch.empty_like(t) for t in (x, r)]
    p[0].grad = torch._neg_view(x.neg())                             # x again
    clip_grad_norm_(p, 1e9, out=out)
    assert torch.equal(out[0], p[0].grad) and torch.equal(out[1], p[1].grad)
    with pytest.raises(ValueError):
        clip_grad_norm_(p, 1.0, out=[torch._neg_view(out[0]), out[1]])
