"""Layer norm, linear layer and gradient clipping against their formulas in float64, element by element.

Tolerances are bounds, derived per element: half a step of the output's type (eps / 2 of the value) plus the float32 work in
front of it. A float32 sum of n terms in any order is off by at most (n - 1) u sum |terms| with u = 2^-24; the kernels' sums are
trees over short runs, so `DEPTH` additions stand for the longest chain a term passes through."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
TYPES = [F32, BF, HF]


def half_step(t):
    """Half a rounding step relative to the value; float16 results below 2^-14 step by 2^-24, bfloat16 and float32 ones below
    2^-126 by far less than any tolerance here."""
    return torch.finfo(t).eps / 2


def floor_of(t):
    return 2.0 ** -25 if t == HF else 2.0 ** -149


def randn(shape, seed, dtype=F32, scale=1.0, shift=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale + shift).to(dtype)


def close(got, want, tol, what):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got.double() - want).abs() <= tol)
    assert not bool(bad.any()), (what, int(bad.sum()), float(((got.double() - want).abs() / tol).nan_to_num(9e9).max()))


# ---- layer norm --------------------------------------------------------------------------------------------------------

def ln_formula(x, w, b, eps, dy=None):
    x = x.double()
    n = x.shape[-1]
    w = torch.ones(n, dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros(n, dtype=torch.float64, device=x.device) if b is None else b.double()
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / ((x - mean).square().mean(-1, keepdim=True) + eps).sqrt()
    xh = (x - mean) * rstd
    out = {"y": xh * w + b, "xh": xh, "rstd": rstd, "w": w, "b": b}
    if dy is not None:
        dy = dy.double()
        g = dy * w
        out["dx"] = rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
        red = tuple(range(x.dim() - 1))
        out["dw"], out["db"] = (dy * xh).sum(red), dy.sum(red)
    return out


def ln_bounds(f, x, dy, t, pt):
    """DEPTH: a thread adds at most 32 elements of a row, then 10 levels of lanes and waves; mean and rstd add a few more."""
    depth = 64 * U
    big = x.double().abs().amax(-1, keepdim=True) * f["rstd"]          # what an error of the mean is multiplied by
    slack = depth * (big + f["xh"].abs() + 1)                          # error of xhat
    out = {"y": half_step(t) * f["y"].abs() + slack * f["w"].abs() + 4 * U * f["b"].abs() + floor_of(t)}
    if dy is not None:
        dy = dy.double().abs()
        g = dy * f["w"].abs()
        part = (g * (f["xh"].abs() + slack)).mean(-1, keepdim=True)
        out["dx"] = (half_step(t) * f["dx"].abs() + floor_of(t)
                     + f["rstd"] * (depth * (g + g.mean(-1, keepdim=True) + f["xh"].abs() * part + g * f["xh"].abs())
                                    + slack * part + f["xh"].abs() * (g * slack).mean(-1, keepdim=True)))
        red = tuple(range(dy.dim() - 1))
        rows = dy.numel() // dy.shape[-1]
        chain = (min(rows, 160) + 64) * U                              # rows of one slot, then the partial rows
        out["dw"] = half_step(pt) * f["dw"].abs() + (dy * (chain * f["xh"].abs() + slack)).sum(red) + floor_of(pt)
        out["db"] = half_step(pt) * f["db"].abs() + chain * dy.sum(red) + floor_of(pt)
    return out


def check_ln(x, w, b, dy, eps=1e-5):
    from diffusion_model_nemo_amd.modules import layer_norm
    t, pt = x.dtype, (w if w is not None else b).dtype if (w is not None or b is not None) else x.dtype
    f = ln_formula(x, w, b, eps, dy)
    tol = ln_bounds(f, x, dy, t, pt)
    with torch.no_grad():
        y0 = layer_norm(x, w, b, eps)
    leaves = [v.detach().requires_grad_(True) for v in (x, w, b) if v is not None]
    it = iter(leaves)
    args = [next(it) if v is not None else None for v in (x, w, b)]
    y = layer_norm(*args, eps)
    assert torch.equal(y, y0) and y.dtype == t and y.is_contiguous()
    close(y, f["y"], tol["y"], "y")
    grads = iter(torch.autograd.grad(y, leaves, dy))
    for name, v in (("dx", x), ("dw", w), ("db", b)):
        if v is not None:
            got = next(grads)
            assert got.dtype == v.dtype
            close(got, f[name], tol[name], name)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("width", [1, 2, 7, 8, 63, 64, 65, 100, 128, 250, 256, 511, 512, 1000, 1024, 1111, 2048, 2049, 4096, 4099,
                                   8192, 8200, 16384, 16387, 33001])
def test_layer_norm_widths(dtype, width):
    rows = 37 if width < 5000 else 5
    x = randn((rows, width), 1, dtype, 1.5, 0.3)
    check_ln(x, randn((width,), 2, dtype, 0.1, 1.0), randn((width,), 3, dtype, 0.1), randn((rows, width), 4, dtype))


@pytest.mark.parametrize("rows", [1, 2, 31, 1025, 5003])
@pytest.mark.parametrize("width", [24, 130, 768, 4096])
def test_layer_norm_rows_with_float32_parameters(rows, width):
    x = randn((rows, width), 5, BF, 2.0, -1.0)
    check_ln(x, randn((width,), 6, F32, 0.1, 1.0), randn((width,), 7, F32, 0.1), randn((rows, width), 8, BF))


def test_layer_norm_without_parameters_and_with_one_of_them():
    x, dy = randn((9, 200), 1, HF), randn((9, 200), 2, HF)
    check_ln(x, None, None, dy)
    check_ln(x, randn((200,), 3, F32, 0.1, 1.0), None, dy)
    check_ln(x, None, randn((200,), 3, HF), dy)


def test_layer_norm_offset_constant_and_extreme_rows():
    x = randn((8, 1000), 1, F32, 1.0, 1000.0)
    x[1] = 5.0                       # no variance: xhat = 0
    x[2] *= 1e-20
    x[3] = randn((1000,), 2) * 1e15
    check_ln(x, randn((1000,), 3), randn((1000,), 4), randn((8, 1000), 5))


def test_layer_norm_nonfinite_rows_stay_in_their_rows():
    from diffusion_model_nemo_amd.modules import layer_norm
    x = randn((6, 130), 1, BF)
    clean = layer_norm(x)
    x[1, 3], x[2, 7], x[4, 129] = float("nan"), float("inf"), float("-inf")
    y = layer_norm(x)
    for r in range(6):
        if r in (1, 2, 4):
            assert bool(torch.isnan(y[r, 3 if r == 1 else 0])), r
        else:
            assert torch.equal(y[r], clean[r])


def test_layer_norm_strides_shapes_and_expanded_gradients():
    from diffusion_model_nemo_amd.modules import layer_norm
    w, b = randn((96,), 1, F32, 0.1, 1.0), randn((96,), 2, F32)
    big = randn((40, 200), 3, BF)
    check_ln(big[:, 5:101], w, b, randn((40, 200), 4, BF)[:, 50:146])       # rows 200 apart, no 16-byte boundary
    check_ln(randn((96, 40), 5, BF).t(), w, b, randn((40, 96), 6, BF))      # transposed: copied
    check_ln(randn((2, 3, 5, 96), 7, BF), w, b, randn((2, 3, 5, 96), 8, BF))
    check_ln(randn((96,), 9, BF).expand(7, 96), w, b, randn((7, 96), 10, BF))
    check_ln(randn((1, 96), 9, BF).expand(7, 96).t()[:, :1].t(), w, b, randn((1, 96), 10, BF))
    x = randn((4, 96), 11, BF).requires_grad_(True)
    (g,) = torch.autograd.grad(layer_norm(x, w, b).sum(), x)                # the gradient of a sum is one expanded element
    f = ln_formula(x.detach(), w, b, 1e-5, torch.ones(4, 96, device="cuda"))
    close(g, f["dx"], ln_bounds(f, x.detach(), torch.ones(4, 96, device="cuda"), BF, F32)["dx"], "dx")


def test_layer_norm_empty_batch():
    from diffusion_model_nemo_amd.modules import layer_norm
    x, w, b = (v.requires_grad_(True) for v in (randn((0, 33), 1), randn((33,), 2), randn((33,), 3)))
    y = layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty(0, 33, device="cuda"))
    assert y.shape == dx.shape == (0, 33) and not dw.any() and not db.any()


def test_layer_norm_gradient_agrees_with_differences():
    from diffusion_model_nemo_amd.modules import layer_norm
    x, w, b, dy = randn((3, 17), 1), randn((17,), 2), randn((17,), 3), randn((3, 17), 4)
    leaves = [v.clone().requires_grad_(True) for v in (x, w, b)]
    grads = torch.autograd.grad(layer_norm(*leaves), leaves, dy)
    h = 2.0 ** -7
    for which, (leaf, grad) in enumerate(zip((x, w, b), grads)):
        v = randn(leaf.shape, 20 + which)
        ends = []
        for s in (h, -h):
            args = [x, w, b]
            args[which] = leaf + s * v
            ends.append((layer_norm(*args).double() * dy.double()).sum())
        slope = float((ends[0] - ends[1]) / (2 * h))
        want = float((grad.double() * v.double()).sum())
        # rounding of the two values over the step, and the third derivative's h^2 / 6 (of order one here, times 17 * 3 terms)
        assert abs(slope - want) <= 64 * U * float(dy.abs().sum()) * 8 / h + h * h * float((dy.abs().sum())) * 8, (which, slope, want)


def test_layer_norm_same_bits_again_on_another_stream_and_in_a_graph():
    from diffusion_model_nemo_amd.modules import layer_norm
    x, w, b = (v.requires_grad_(True) for v in (randn((300, 520), 1, BF), randn((520,), 2, F32), randn((520,), 3, F32)))
    dy = randn((300, 520), 4, BF)

    def step():
        y = layer_norm(x, w, b)
        return (y.detach(),) + torch.autograd.grad(y, (x, w, b), dy)

    want = step()
    assert all(torch.equal(p, q) for p, q in zip(step(), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(other, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for turn in range(3):
        with torch.no_grad():
            x.copy_(randn((300, 520), 10 + turn, BF))
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, eager)), turn


# ---- linear layer ------------------------------------------------------------------------------------------------------

def act_formula(z, kind):
    if kind == "relu":
        return z.clamp(min=0), (z > 0).double()
    if kind == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if kind == "gelu":
        cdf = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return z, torch.ones_like(z)


def product(a, b):
    """a b and |a| |b| in float64 (operands laid out plainly)."""
    a, b = a.double().contiguous(), b.double().contiguous()
    return a @ b, a.abs() @ b.abs()


def check_linear(x, w, b, r, kind, dy=None):
    """Bounds: a float32 sum of k products is off by at most (k + splits) u sum |products| in any order; the matrix cores add
    k one after the other within a split, so k u is the bound that holds for every split. The activations' slopes are at most
    1.13 and their curvature at most 1.2; `1.2e-6` is the relative error of the float32 / 16-bit tail fits with the hardware
    exponential and reciprocal (an argument of exp up to 14 in size is off by 14 u, each function by an ulp)."""
    from diffusion_model_nemo_amd.modules import linear
    t = x.dtype
    x2, k, n = x.reshape(-1, x.shape[-1]), x.shape[-1], w.shape[0]
    z, za = product(x2, w.t())
    ez = (k + 64) * U * za
    if b is not None:
        z = z + b.double()
        ez = ez + 4 * U * (z.abs() + b.double().abs())
    a, slope = act_formula(z, kind)
    want = a + (0 if r is None else r.reshape(-1, n).double())
    tol = half_step(t) * want.abs() + 1.13 * ez + 2.4e-6 * a.abs() + 4 * U * (a.abs() + want.abs()) + floor_of(t)
    with torch.no_grad():
        y0 = linear(x, w, b, kind, r)
    assert y0.dtype == t and y0.is_contiguous() and y0.shape == x.shape[:-1] + (n,)
    close(y0.reshape(-1, n), want, tol, "y")
    if dy is None:
        return
    names = [("x", x), ("w", w), ("b", b), ("r", r)]
    leaves = {m: v.detach().requires_grad_(True) for m, v in names if v is not None}
    y = linear(leaves["x"], leaves["w"], leaves.get("b"), kind, leaves.get("r"))
    assert torch.equal(y, y0)
    got = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))
    d2 = dy.reshape(-1, n).double()
    dz = d2 * slope
    # z is kept rounded (half a step of z times the slope's own slope), the sums are off by ez, dz is rounded for the products
    edz = torch.zeros_like(dz)
    if kind is not None:
        edz = d2.abs() * (1.2 * (half_step(t) * z.abs() + ez + floor_of(t)) + 4e-6 + 4 * U)
        if kind == "relu":   # the slope jumps at 0: only values whose sign is in doubt can change, and they by all of dy
            edz = torch.where(z.abs() <= ez + floor_of(t), d2.abs(), torch.zeros_like(dz))
    edz_op = edz + (half_step(t) * (dz.abs() + edz) + floor_of(t) if kind is not None else 0)
    rows = d2.shape[0]
    for name, (want, size), err, depth in (
            ("x", product(dz, w), edz_op @ w.double().abs(), n),
            ("w", product(dz.t(), x2), edz_op.t().contiguous() @ x2.double().abs(), rows)):
        size = size + err
        g = got[name].reshape(want.shape)
        assert got[name].dtype == t
        close(g, want, half_step(t) * want.abs() + err + (depth + 64) * U * size + floor_of(t), "d" + name)
    if b is not None:
        want = dz.sum(0)
        close(got["b"], want, half_step(t) * want.abs() + edz.sum(0) + (rows + 64) * U * (dz.abs() + edz).sum(0) + floor_of(t), "db")
    if r is not None:
        assert torch.equal(got["r"], dy)


def linear_case(m, k, n, dtype, kind, bias, res, train=True, seed=0):
    x, w = randn((m, k), seed + 1, dtype), randn((n, k), seed + 2, dtype, k ** -0.5)
    b = randn((n,), seed + 3, dtype, 0.3) if bias else None
    r = randn((m, n), seed + 4, dtype) if res else None
    check_linear(x, w, b, r, kind, randn((m, n), seed + 5, dtype) if train else None)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 8, 8), (2, 3, 5), (1, 64, 64), (16, 32, 16), (17, 40, 24), (64, 64, 64), (65, 72, 80),
                                   (63, 65, 61), (128, 128, 128), (129, 136, 144), (130, 127, 131), (200, 512, 96), (31, 1000, 153),
                                   (5, 2056, 33), (300, 24, 520), (1000, 8, 7), (257, 260, 4)])
def test_linear_sizes(dtype, m, k, n):
    linear_case(m, k, n, dtype, "gelu", True, True)
    linear_case(m, k, n, dtype, None, True, False, seed=10)


@pytest.mark.parametrize("kind", [None, "relu", "silu", "gelu"])
@pytest.mark.parametrize("bias,res", [(False, False), (True, False), (False, True), (True, True)])
def test_linear_epilogues(kind, bias, res):
    for dtype in TYPES:
        linear_case(70, 96, 104, dtype, kind, bias, res)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m", [1, 2, 3, 4, 7, 8, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65])
def test_linear_few_rows(dtype, m):
    linear_case(m, 1024, 272, dtype, "silu", True, True, train=False)
    linear_case(m, 999, 77, dtype, "gelu", True, False, train=False, seed=20)


@pytest.mark.parametrize("m,k,n", [(2048, 2048, 2048), (1555, 1032, 2056), (4001, 520, 264), (64, 8192, 128), (256, 4096, 256)])
def test_linear_large_and_split_products(m, k, n):
    linear_case(m, k, n, BF, "gelu", True, True)
    linear_case(m, k, n, HF, None, True, False, seed=30)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,k,n", [(4096, 320, 1280), (64, 1024, 1024), (2047, 1021, 1030), (6000, 1024, 1000), (8192, 128, 512), (256, 320, 320)])
def test_linear_backward_products_beside_each_other(dtype, m, k, n):
    """dx and dW from one launch: either's k split, odd sizes, either's tiles in front."""
    linear_case(m, k, n, dtype, "silu", True, False, seed=60)


def test_linear_float32_large():
    linear_case(1555, 1032, 520, F32, "silu", True, True)
    linear_case(4096, 64, 256, F32, "gelu", True, False)
    linear_case(100, 3, 4096, F32, None, False, False)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_linear_strides_and_shapes(dtype):
    w, b = randn((80, 72), 1, dtype, 0.1), randn((80,), 2, dtype)
    big, rbig = randn((50, 200), 3, dtype), randn((50, 120), 4, dtype)
    dy = randn((50, 200), 5, dtype)
    check_linear(big[:, 8:80], w, b, rbig[:, 40:], "gelu", dy[:, 16:96])     # rows apart, on 16-byte boundaries
    check_linear(big[:, 3:75], w, b, rbig[:, 39:119], "gelu", dy[:, 5:85])   # ... and off them
    check_linear(randn((72, 50), 6, dtype).t(), w, b, None, None, randn((80, 50), 7, dtype).t())
    check_linear(randn((2, 5, 3, 72), 8, dtype), w, b, randn((2, 5, 3, 80), 9, dtype), "silu", randn((2, 5, 3, 80), 10, dtype))
    check_linear(randn((72,), 11, dtype), w, b, None, "relu", randn((80,), 12, dtype))
    check_linear(randn((72,), 11, dtype).expand(9, 72), w.t().contiguous().t(), b, None, None, randn((1,), 12, dtype).expand(9, 80))


def test_linear_activation_tails_and_nonfinite_rows():
    from diffusion_model_nemo_amd.modules import linear
    one = torch.ones(1, 1, device="cuda")
    z = torch.cat([torch.linspace(-14, 14, 4001), torch.tensor([0.0, -0.0, 50.0, -50.0, 100.0, -100.0, 1e-30, -1e-30])]).cuda().view(-1, 1)
    for kind in ("relu", "silu", "gelu"):
        y = linear(z, one, activation=kind)
        want, slope = act_formula(z.double(), kind)
        # exp's argument z^2 / 2 is rounded (98 u at 14), everything else by a few ulps
        close(y, want, 1e-5 * want.abs() + 1e-37, kind)
        x = z.clone().requires_grad_(True)
        (g,) = torch.autograd.grad(linear(x, one, activation=kind), x, torch.ones_like(z))
        close(g, slope, 1e-5 * slope.abs() + 4e-6 * torch.exp(-z.double().square() / 4) + 1e-30, "slope of " + kind)
    for dtype in TYPES:
        x, w = randn((40, 64), 1, dtype), randn((48, 64), 2, dtype)
        clean = linear(x, w, activation="gelu")
        x[3, 5], x[20, 63], x[39, 0] = float("nan"), float("inf"), float("-inf")
        y = linear(x, w, activation="gelu")
        assert bool(torch.isnan(y[3]).all()) and not bool(torch.isfinite(y[20]).all()) and not bool(torch.isfinite(y[39]).all())
        rest = [i for i in range(40) if i not in (3, 20, 39)]
        assert torch.equal(y[rest], clean[rest])
        assert bool(torch.isnan(linear(x, w, activation="relu")[3]).all())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("kind", [None, "gelu"])
def test_linear_gradients_asked_for_one_by_one(kind, dtype):
    from diffusion_model_nemo_amd.modules import linear
    for shape in ((70, 96, 104), (33, 45, 51)):
        m, k, n = shape
        args = [randn((m, k), 1, dtype), randn((n, k), 2, dtype, k ** -0.5), randn((n,), 3, dtype), randn((m, n), 4, dtype)]
        dy = randn((m, n), 5, dtype)
        every = [a.clone().requires_grad_(True) for a in args]
        want = torch.autograd.grad(linear(every[0], every[1], every[2], kind, every[3]), every, dy)
        for i in range(4):
            some = [a.clone().requires_grad_(i == j) for j, a in enumerate(args)]
            (got,) = torch.autograd.grad(linear(some[0], some[1], some[2], kind, some[3]), some[i], dy)
            assert torch.equal(got, want[i]), (shape, i)


@pytest.mark.parametrize("kind", [None, "gelu"])
def test_linear_rows_a_million_elements_apart(kind):
    """Views of a tensor with very long rows: x, the residual and the incoming gradient."""
    from diffusion_model_nemo_amd.modules import linear
    wide = randn((3, (1 << 20) + 72), 1, BF)
    w, b = randn((48, 64), 2, BF, 0.125), randn((48,), 3, BF)
    x, r, dy = wide[:, 8:72], wide[:, 100:148], wide[:, 1000:1048]
    got = []
    for at, rt, dt in ((x, r, dy), (x.contiguous(), r.contiguous(), dy.contiguous())):
        leaves = [t.detach().requires_grad_(True) for t in (at, w, b, rt)]
        y = linear(leaves[0], leaves[1], leaves[2], kind, leaves[3])
        got.append((y,) + torch.autograd.grad(y, leaves, dt))
    assert all(torch.equal(p, q) for p, q in zip(*got))


def test_elements_behind_the_two_thousand_millionth():
    """More than 2^31 elements in a tensor: the rows at its end, and sums that only rows at both ends feed."""
    from diffusion_model_nemo_amd.modules import layer_norm, linear
    from diffusion_model_nemo_amd.training import clip_grad_norm_
    rows, n, k, ends = (1 << 20) + 3, 2056, 64, 40
    at = torch.cat([torch.arange(ends, device="cuda"), torch.arange(rows - ends, rows, device="cuda")])
    big = torch.zeros(rows, n, dtype=BF, device="cuda")
    big[at] = randn((2 * ends, n), 1, BF)
    dy = torch.zeros_like(big)
    dy[at] = randn((2 * ends, n), 2, BF)
    w, b = randn((n,), 3, BF, 0.1, 1.0), randn((n,), 4, BF)
    leaves = [t.requires_grad_(True) for t in (big, w, b)]
    y = layer_norm(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    f = ln_formula(big[at].detach(), w.detach(), b.detach(), 1e-5, dy[at])
    tol = ln_bounds(f, big[at].detach(), dy[at], BF, BF)
    for name, got in (("y", y[at]), ("dx", grads[0][at]), ("dw", grads[1]), ("db", grads[2])):
        close(got, f[name], tol[name], name)
    assert not bool(grads[0][ends:rows - ends].any())
    del y, grads, leaves
    big = big.detach()

    x, weight = randn((rows, k), 5, BF), randn((n, k), 6, BF, 0.125)
    leaves = [x.requires_grad_(True), weight.requires_grad_(True)]
    y = linear(*leaves, None, None, big)
    xs, ds, wd = x.detach()[at], dy[at], weight.detach()
    want, size = product(xs, wd.t())
    want = want + big[at].double()
    close(y[at], want, half_step(BF) * want.abs() + (k + 64) * U * (size + want.abs()) + floor_of(BF), "y")
    dx, dw = torch.autograd.grad(y, leaves, dy)
    del y
    for got, (want, size), depth in ((dx[at], product(ds, wd), n), (dw, product(ds.t(), xs), 2 * ends)):
        close(got, want, half_step(BF) * want.abs() + (depth + 64) * U * size + floor_of(BF), "dx, dw")
    assert not bool(dx[ends:rows - ends].any())
    del dx, dw, big

    p = torch.nn.Parameter(torch.zeros(rows, n, dtype=BF, device="cuda"))
    p.grad = dy
    before = dy[at].clone()
    norm = clip_grad_norm_(p, 1.0)
    want = before.double().square().sum().sqrt()
    assert abs(float(norm) - float(want)) <= 4 * U * float(want)
    close(dy[at], before.double() / (want + 1e-6), (half_step(BF) + 4 * U) * (before.double() / want).abs() + floor_of(BF), "clipped")


def test_linear_and_layer_norm_shared_repeated_and_interleaved_uses():
    """One tensor as input and residual, one weight twice, a graph walked twice, recomputation, an input changed behind the
    forward's back, two streams at once: all in bits, against the calls one by one."""
    from torch.utils.checkpoint import checkpoint
    from diffusion_model_nemo_amd.modules import layer_norm, linear
    x, w, b = randn((777, 320), 1, BF), randn((320, 320), 2, BF, 0.05), randn((320,), 3, BF)
    dy = randn((777, 320), 4, BF)

    def step(x, w, b, r):
        leaves = [t.detach().clone().requires_grad_(True) for t in (x, w, b, r)]
        y = linear(layer_norm(leaves[0], None, leaves[2]), leaves[1], leaves[2], "gelu", leaves[3])
        return (y.detach(),) + torch.autograd.grad(y, leaves, dy)

    def plain(x, w, b, r):
        leaves = [t.detach().clone().requires_grad_(True) for t in (x, w, b, r)]
        y = linear(*leaves[:3], "gelu", leaves[3])
        return (y.detach(),) + torch.autograd.grad(y, leaves, dy)

    one = plain(x, w, b, x)
    xs, ws, bs = (t.detach().clone().requires_grad_(True) for t in (x, w, b))
    y = linear(xs, ws, bs, "gelu", xs)
    assert torch.equal(y, one[0])
    for _ in range(2):   # the same graph twice, the same bits
        gx, gw, gb = torch.autograd.grad(y, (xs, ws, bs), dy, retain_graph=True)
        assert torch.equal(gx, one[1] + one[4]) and torch.equal(gw, one[2]) and torch.equal(gb, one[3])

    first = linear(xs, ws)                      # one weight in two layers: the sum of both layers' gradients
    gx, gw = torch.autograd.grad(linear(first, ws), (xs, ws), dy)
    f1, w1, x1, w2 = (t.detach().requires_grad_(True) for t in (first, w, x, w))
    gf, gw2 = torch.autograd.grad(linear(f1, w2), (f1, w2), dy)
    gx1, gw1 = torch.autograd.grad(linear(x1, w1), (x1, w1), gf)
    assert torch.equal(gx, gx1) and torch.equal(gw, gw2 + gw1)

    xc = x.detach().requires_grad_(True)
    yc = checkpoint(lambda t: linear(t, w, b, "gelu", t), xc, use_reentrant=False)
    assert torch.equal(yc, one[0])
    xr = x.detach().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(yc, xc, dy)[0], torch.autograd.grad(linear(xr, w, b, "gelu", xr), xr, dy)[0])

    h = x.detach().clone()
    y = linear(h, ws, bs, "relu")
    h.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, ws, dy)

    want = step(x, w, b, x)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(6):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(step(x, w, b, x))
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for r in got for p, q in zip(r, want))


def test_linear_empty_batch():
    from diffusion_model_nemo_amd.modules import linear
    for kind in (None, "gelu"):
        x, w, b = (v.requires_grad_(True) for v in (randn((0, 24), 1, BF), randn((16, 24), 2, BF), randn((16,), 3, BF)))
        y = linear(x, w, b, kind)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty((0, 16), dtype=BF, device="cuda"))
        assert y.shape == (0, 16) and dx.shape == (0, 24) and not dw.any() and not db.any()


def test_linear_refusals():
    from diffusion_model_nemo_amd.modules import Linear, linear
    x, w = randn((4, 8), 1), randn((6, 8), 2)
    for args in ((x, randn((6, 7), 3)), (x, w, randn((5,), 3)), (x, w.bfloat16()), (x, w, None, "tanh"),
                 (x, w, None, None, randn((4, 5), 3)), (x, w, None, None, randn((6,), 3)), (x.double(), w.double()),
                 (x, randn((0, 8), 3)), (x, randn((8,), 3))):
        with pytest.raises(ValueError):
            linear(*args)
    with pytest.raises(RuntimeError):
        linear(x, w.cpu())
    with pytest.raises(ValueError):
        Linear(8, 6, activation="tanh")
    p = x.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(linear(p, w, activation="silu").sum(), p, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()          # the backward pass is not differentiable


@pytest.mark.parametrize("kind", [None, "silu", "gelu"])
def test_linear_gradient_agrees_with_differences(kind):
    from diffusion_model_nemo_amd.modules import linear
    parts = {"x": randn((5, 12), 1), "w": randn((9, 12), 2, scale=0.3), "b": randn((9,), 3), "r": randn((5, 9), 4)}
    dy = randn((5, 9), 5)
    leaves = {k: v.clone().requires_grad_(True) for k, v in parts.items()}
    y = linear(leaves["x"], leaves["w"], leaves["b"], kind, leaves["r"])
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))
    h = 2.0 ** -7
    for i, (name, v) in enumerate(parts.items()):
        way = randn(v.shape, 20 + i)
        way /= way.abs().max()
        ends = []
        for s in (h, -h):
            p = dict(parts)
            p[name] = v + s * way
            ends.append((linear(p["x"], p["w"], p["b"], kind, p["r"]).double() * dy.double()).sum())
        slope, want = float((ends[0] - ends[1]) / (2 * h)), float((grads[name].double() * way.double()).sum())
        # the values' rounding over the step; the third derivative (at most 2.4) times h^2 / 6 times the inputs' sizes cubed
        reach = float((parts["x"].abs().sum(1).max() + 1) ** 3 * dy.abs().sum())
        assert abs(slope - want) <= 64 * U * 20 * float(dy.abs().sum()) / h + 0.4 * h * h * reach, (name, slope, want)


# ---- the operators together -----------------------------------------------------------------------------------------------

def test_block_trains_with_clipping_in_eager_mode_and_in_a_graph():
    """x + W2 gelu(W1 norm(x) + b1) + b2, its gradients against float64 autograd, clipped together; then the same step recorded
    and replayed on new inputs."""
    from diffusion_model_nemo_amd.modules import LayerNorm, Linear
    from diffusion_model_nemo_amd.training import clip_grad_norm_
    torch.manual_seed(0)
    norm, up, down = LayerNorm(136).cuda(), Linear(136, 544, activation="gelu").cuda(), Linear(544, 136).cuda()
    params = [p for m in (norm, up, down) for p in m.parameters()]
    x, dy = randn((203, 136), 1), randn((203, 136), 2)
    out = [torch.zeros_like(p) for p in params]

    def step():
        for p in params:
            p.grad = None
        y = down(up(norm(x)), residual=x)
        for p, g in zip(params, torch.autograd.grad(y, params, dy)):
            p.grad = g
        return y.detach(), clip_grad_norm_(params, 5.0, out=out)

    y, total = step()
    ref = [p.detach().double().requires_grad_(True) for p in params]
    n, w1, b1, w2, b2 = None, ref[2], ref[3], ref[4], ref[5]
    n = torch.nn.functional.layer_norm(x.double(), (136,), ref[0], ref[1])
    want_y = torch.nn.functional.gelu(n @ w1.t() + b1) @ w2.t() + b2 + x.double()
    grads, want_y = torch.autograd.grad(want_y, ref, dy.double()), want_y.detach()
    want_total, want = clip_formula(grads, 5.0, 2.0)
    # float32 sums of up to 544 products and 203 rows: a few hundred u of values of order one to ten
    assert float((y.double() - want_y).abs().max()) <= 1000 * U * 8
    assert float(want_total) > 5.0 and abs(float(total) - float(want_total)) <= 1000 * U * float(want_total)
    for o, w in zip(out, want):
        assert float((o.double() - w).abs().max()) <= 1000 * U * float(w.abs().max() + 1)
    for p in params:
        p.grad = None
    del y, total
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for turn in range(3):
        x.copy_(randn((203, 136), 40 + turn))
        graph.replay()
        kept = [got[0].clone(), got[1].clone()] + [o.clone() for o in out]
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip([eager[0], eager[1]] + out, kept)), turn


def test_capture_beside_a_living_eager_graph_is_refused_and_large_products_are_captured():
    from diffusion_model_nemo_amd.modules import layer_norm, linear
    x = randn((2100, 1032), 1, BF).requires_grad_(True)
    w, b = randn((2056, 1032), 2, BF, 0.03).requires_grad_(True), randn((2056,), 3, BF).requires_grad_(True)
    dy = randn((2100, 2056), 4, BF)
    alive = linear(x, w, b, "gelu")
    for call in (lambda: linear(x, w, b, "gelu"), lambda: layer_norm(x)):
        with pytest.raises(RuntimeError, match="still lives"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
    want = alive.detach().clone()
    del alive

    def step():
        y = linear(x, w, b, "gelu")
        y.backward(dy)
        return y.detach()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(step(), want)
    torch.cuda.current_stream().wait_stream(side)
    for p in (x, w, b):
        p.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    grads = [p.grad for p in (x, w, b)]          # the graph's own, overwritten by every replay
    for turn in range(3):
        with torch.no_grad():
            x.copy_(randn((2100, 1032), 20 + turn, BF))
        graph.replay()
        kept = [got.clone()] + [g.clone() for g in grads]
        y = linear(x, w, b, "gelu")
        eager = torch.autograd.grad(y, (x, w, b), dy)
        torch.cuda.synchronize()
        assert torch.equal(kept[0], y.detach()) and all(torch.equal(p, q) for p, q in zip(kept[1:], eager)), turn
        del y, eager


# ---- gradient clipping -----------------------------------------------------------------------------------------------------

def params_with(grads):
    out = []
    for g in grads:
        p = torch.nn.Parameter(torch.empty(g.shape, dtype=g.dtype, device=g.device))
        p.grad = g
        out.append(p)
    return out


def clip_formula(grads, max_norm, kind, scale=1.0):
    flat = [g.double().flatten() * scale for g in grads]
    flat = [f for f in flat if f.numel()]
    if kind == math.inf:
        norm = torch.stack([f.abs().max() for f in flat]).max()
    else:
        norm = torch.stack([f.square().sum() for f in flat]).sum().sqrt()
    c = (max_norm / (norm + 1e-6)).clamp(max=1.0)
    return norm, [g.double() * scale * c for g in grads]


SHAPES = [(1,), (3,), (64, 32, 3, 3), (17, 5), (), (0, 4), (8191,), (8193,), (257, 129), (2, 1), (33000,)]


@pytest.mark.parametrize("kind", [2.0, math.inf], ids=["two", "inf"])
@pytest.mark.parametrize("clipped", [False, True], ids=["within", "clipped"])
@pytest.mark.parametrize("dtypes", [(F32,), (BF,), (HF,), (F32, BF, HF)], ids=["fp32", "bf16", "fp16", "mixed"])
def test_clip_many_tensors(dtypes, clipped, kind):
    from diffusion_model_nemo_amd.training import clip_grad_norm_
    grads = [randn(s, 30 + i, dtypes[i % len(dtypes)], 0.1 * (1 + i % 3)) for i, s in enumerate(SHAPES * 40)]   # 440: several launches
    norm0, _ = clip_formula(grads, 1.0, kind)
    limit = float(norm0) * (0.37 if clipped else 3.0)
    norm, want = clip_formula(grads, limit, kind)
    params = params_with([g.clone() for g in grads])
    got = clip_grad_norm_(params, limit, norm_type=kind)
    # the squares are added in float64; what is left are the norm's own rounding, the limit's and the factor's
    assert got.shape == () and got.dtype == F32 and abs(float(got) - float(norm)) <= 2 * U * float(norm)
    for p, g, w in zip(params, grads, want):
        if not clipped:
            assert torch.equal(p.grad, g)
        else:
            close(p.grad, w, (half_step(g.dtype) + 3 * U) * w.abs() + floor_of(g.dtype), "grad")


@pytest.mark.parametrize("to", TYPES, ids=str)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_clip_into_other_tensors_with_a_scale(dtype, to):
    from diffusion_model_nemo_amd.training import clip_grad_norm_
    grads = [randn(s, 50 + i, dtype, 0.2) for i, s in enumerate(SHAPES)]
    norm, want = clip_formula(grads, 0.9, 2.0, 0.125)
    before = [g.clone() for g in grads]
    out = [torch.full(g.shape, float("nan"), dtype=to, device="cuda") for g in grads]
    got = clip_grad_norm_(params_with(grads), 0.9, grad_scale=0.125, out=out)
    assert abs(float(got) - float(norm)) <= 2 * U * float(norm)
    for g, b, o, w in zip(grads, before, out, want):
        assert torch.equal(g, b)
        close(o, w, (half_step(to) + 3 * U) * w.abs() + floor_of(to), "out")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_clip_tightly_packed_views_leave_their_neighbours_alone(dtype):
    from diffusion_model_nemo_amd.training import clip_grad_norm_
    flat = randn((60000,), 1, dtype)
    keep = flat.clone()
    cuts, at = [], 1
    for n in (1, 2, 3, 5, 7, 8, 9, 31, 33, 8192, 8193, 16385, 20001):
        cuts.append((at, at + n))
        at += n + (n % 2)
    params = params_with([flat[a:b] for a, b in cuts])
    norm, want = clip_formula([keep[a:b] for a, b in cuts], 1.0, 2.0)
    clip_grad_norm_(params, 1.0)
    mask = torch.ones(60000, dtype=torch.bool, device="cuda")
    for (a, b), w in zip(cuts, want):
        close(flat[a:b], w, (half_step(dtype) + 3 * U) * w.abs() + floor_of(dtype), (a, b))
        mask[a:b] = False
    assert torch.equal(flat[mask], keep[mask])


def test_clip_extreme_values_and_nonfinite_gradients():
    from diffusion_model_nemo_amd.training import clip_grad_norm_
    big = params_with([torch.full((1000,), 1e30, device="cuda"), torch.full((10,), 1e-30, device="cuda")])
    assert abs(float(clip_grad_norm_(big, math.inf)) / (1e30 * math.sqrt(1000)) - 1) < 1e-6     # squares overflow float32
    small = params_with([torch.full((100,), 1e-30, device="cuda")])
    assert abs(float(clip_grad_norm_(small, 1.0)) / 1e-29 - 1) < 1e-6                             # ... and underflow it
    for bad, kind in ((float("nan"), 2.0), (float("nan"), math.inf), (float("inf"), 2.0), (float("-inf"), math.inf)):
        for at in (0, 4999, 9999):
            g = randn((10000,), 3)
            g[at] = bad
            params = params_with([randn((5,), 4), g])
            first = params[0].grad.clone()
            with pytest.raises(RuntimeError, match="non-finite"):
                clip_grad_norm_(params, 1.0, norm_type=kind, error_if_nonfinite=True)
            assert torch.equal(params[0].grad, first)
            n = clip_grad_norm_(params, 1.0, norm_type=kind)
            assert math.isnan(float(n)) if math.isnan(bad) else float(n) == math.inf
            # as in torch: a NaN norm makes every gradient NaN, an infinite one makes finite gradients zero
            assert bool(torch.isnan(params[0].grad).all()) if math.isnan(bad) else not bool(params[0].grad.any())
            assert bool(torch.isnan(params[1].grad[at]))


def test_clip_scattered_and_reordered_gradients():
    from diffusion_model_nemo_amd.training import clip_grad_norm_
    base = randn((40, 60), 1)
    keep = base.clone()
    perm = randn((4, 6, 5, 7), 2).to(memory_format=torch.channels_last)
    pk = perm.clone()
    norm, want = clip_formula([keep[:, 3:50], pk, keep[:, 55:].t()], 1.0, 2.0)
    got = clip_grad_norm_(params_with([base[:, 3:50], perm, base[:, 55:].t()]), 1.0)
    assert abs(float(got) - float(norm)) <= 2 * U * float(norm)
    for g, w in zip((base[:, 3:50], perm, base[:, 55:].t()), want):
        close(g, w, (half_step(F32) + 3 * U) * w.abs() + 1e-40, "grad")
    assert torch.equal(base[:, :3], keep[:, :3]) and torch.equal(base[:, 50:55], keep[:, 50:55])


def test_clip_skips_parameters_without_gradients_and_handles_none_at_all():
    from diffusion_model_nemo_amd.training import clip_grad_norm_
    p = params_with([randn((10,), 1), randn((20,), 2)])
    p[0].grad = None
    want = float(p[1].grad.double().norm())
    assert abs(float(clip_grad_norm_(p, 1e9)) - want) <= 2 * U * want
    out = [torch.full((10,), 7.0, device="cuda"), torch.zeros(20, device="cuda")]
    clip_grad_norm_(p, 1e9, out=out)
    assert torch.equal(out[1], p[1].grad) and bool((out[0] == 7).all())
    assert float(clip_grad_norm_([], 1.0)) == 0.0
    assert float(clip_grad_norm_(params_with([torch.zeros((0, 3), device="cuda")]), 1.0)) == 0.0
    single = params_with([randn((64,), 3)])[0]
    assert abs(float(clip_grad_norm_(single, 1e9)) - float(single.grad.double().norm())) <= 1e-5


def test_clip_refuses_overlaps_and_bad_arguments():
    from diffusion_model_nemo_amd._native import DmnError
    from diffusion_model_nemo_amd.training import clip_grad_norm_
    g = randn((100,), 1)
    keep = g.clone()
    for grads in ([g, g], [g[:60], g[59:]], [g[10:20], g]):
        with pytest.raises(DmnError, match="overlaps"):
            clip_grad_norm_(params_with(grads), 1.0)
    square = g.view(10, 10)
    for grads in ([square[:, :5], square[:, :5]], [square[:, :5], square[:, 4:]], [square[:, :5], g]):   # scattered ones too
        with pytest.raises(ValueError, match="shares memory"):
            clip_grad_norm_(params_with(grads), 1.0)
    out = torch.zeros(100, device="cuda")
    with pytest.raises(DmnError, match="overlaps"):
        clip_grad_norm_(params_with([g, g]), 1.0, out=[out, out])
    with pytest.raises(DmnError, match="overlaps"):
        clip_grad_norm_(params_with([g[:50]]), 1.0, out=[g[1:51]])
    with pytest.raises(ValueError):
        clip_grad_norm_(params_with([torch.ones(1, device="cuda").expand(5)]), 1.0)
    with pytest.raises(ValueError):
        clip_grad_norm_(params_with([g]), -1.0)
    with pytest.raises(ValueError):
        clip_grad_norm_(params_with([g]), 1.0, out=[])
    with pytest.raises(ValueError):
        clip_grad_norm_(params_with([g]), 1.0, out=[torch.zeros(99, device="cuda")])
    with pytest.raises(ValueError):
        clip_grad_norm_(params_with([g.double()]), 1.0)
    with pytest.raises(NotImplementedError):
        clip_grad_norm_(params_with([g]), 1.0, norm_type=1.0)
    assert torch.equal(g, keep)
    # the same gradient may be READ twice
    a, b = torch.zeros(100, device="cuda"), torch.zeros(100, device="cuda")
    n = clip_grad_norm_(params_with([g, g]), 1e9, out=[a, b])
    assert torch.equal(a, g) and torch.equal(b, g) and abs(float(n) - math.sqrt(2) * float(g.double().norm())) < 1e-4


def test_clip_in_a_graph_and_repeated():
    from diffusion_model_nemo_amd.training import clip_grad_norm_
    grads = [randn((n,), n, BF) for n in (5, 4096, 20000, 33)]
    out = [torch.zeros_like(g, dtype=F32) for g in grads]
    params = params_with(grads)
    clip_grad_norm_(params, 1.0, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_grad_norm_(params, 1.0, out=out)
    for turn in range(3):
        for i, g in enumerate(grads):
            g.copy_(randn(g.shape, 100 * turn + i, BF))
        graph.replay()
        got = [norm.clone()] + [o.clone() for o in out]
        eager = [torch.zeros_like(o) for o in out]
        n2 = clip_grad_norm_(params, 1.0, out=eager)
        torch.cuda.synchronize()
        assert torch.equal(n2, got[0]) and all(torch.equal(p, q) for p, q in zip(eager, got[1:]))


def test_clip_on_the_autograd_route_of_the_denoising_network():
    from diffusion_model_nemo_amd.models import DDPM
    cfg = {"image_size": 32, "timesteps": 10, "channels": 3,
           "diffusion_model": {"_target_": "diffusion_model_nemo.modules.Unet", "input_dim": 32, "dim": 32,
                               "use_convnext": False, "dropout": 0.0, "compute_dtype": "fp32"},
           "sampler": {"_target_": "diffusion_model_nemo.modules.GaussianDiffusion", "timesteps": 10, "schedule_name": "linear"},
           "loss": {"_target_": "diffusion_model_nemo.loss.DiffusionLoss", "loss_type": "l2", "reduction": "mean"},
           "optim": {"name": "adamw"}}
    torch.manual_seed(0)
    m = DDPM(cfg, trainer={"gradient_clip_val": 0.05}).cuda()
    opt = torch.optim.SGD(m.parameters(), lr=1e-3)
    loss = m.training_step({"pixel_values": randn((2, 3, 32, 32), 1)}, t=torch.tensor([1, 7], device="cuda"), noise=randn((2, 3, 32, 32), 2))
    loss.backward()
    grads = [p.grad.clone() for p in m.parameters()]
    norm, want = clip_formula(grads, 0.05, 2.0)
    assert float(norm) > 0.05
    got = m.configure_gradient_clipping(opt)
    assert abs(float(got) - float(norm)) <= 2 * U * float(norm)
    for p, w in zip(m.parameters(), want):
        close(p.grad, w, 4 * U * w.abs() + 1e-40, "grad")
    assert m.configure_gradient_clipping(opt, gradient_clip_val=0.0) is None
    with pytest.raises(NotImplementedError):
        m.configure_gradient_clipping(opt, gradient_clip_algorithm="value")
