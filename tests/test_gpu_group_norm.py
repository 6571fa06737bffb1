"""norm.group_norm_act / GroupNormAct2d against the definition in 64 bits (differentiated by torch on the CPU).

Tolerances follow the formula, U = 2^-24, d additions one after another (d = pixels x channels of a group / 64 + 64 covers any
split over at least 64 lanes and the joining of their sums):
  mean: d U mean|x| =: e0;  var: relative 2 (d + 4) U, plus e0^2;  rstd: half of it, plus 3 U
  xhat: rstd (e0 + U |x - mean|) + |xhat| off(rstd);  u: |gamma| off(xhat) + 3 U (|gamma xhat| + |u|)
  y: 1.1 off(u) (the steepest slope of the activations) + 8 U |y| + half a step of the type
  du: |dy| (0.5 off(u) + 8 U) (|silu''| <= 0.5); where relu's u is within off(u) of 0 its gate may go either way: |dy|
  A = sum du, B = sum du xhat: the terms' own, plus (d + 2) U sum of sizes; sums over groups and images alike
  dx = rstd (gamma du - m1 - xhat m2): products of the above
"""
import pytest
import torch

U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8}


def _act(u, act):
    return {"none": lambda: u, "relu": lambda: torch.relu(u), "silu": lambda: u * torch.sigmoid(u)}[act]()


def _ref(x, w, b, groups, eps, act):
    """x float64 [N, P, C] -> y; plain definition."""
    n, p, c = x.shape
    t = x.view(n, p, groups, c // groups)
    mean = t.mean((1, 3), keepdim=True)
    var = (t - mean).square().mean((1, 3), keepdim=True)
    xhat = ((t - mean) / (var + eps).sqrt()).view(n, p, c)
    return _act(xhat * w + b, act)


def _tolerances(x, w, b, dy, groups, eps, act, dtype):
    n, p, c = x.shape
    k = c // groups
    t = x.view(n, p, groups, k)
    each = lambda s: s.expand(n, p, groups, k).reshape(n, p, c)                                  # noqa: E731
    d = p * k / 64 + 64
    e0 = d * U * t.abs().mean((1, 3), keepdim=True)
    mean = t.mean((1, 3), keepdim=True)
    var = (t - mean).square().mean((1, 3), keepdim=True)
    rstd = (var + eps) ** -0.5
    off_r = (((d + 4) * U * var + e0 * e0) / (var + eps) + 3 * U)                                # relative
    xhat = each((t - mean) * rstd)
    off_x = each(rstd * (e0 + U * (t - mean).abs())) + xhat.abs() * each(off_r)
    u = xhat * w + b
    off_u = w.abs() * off_x + 3 * U * ((w * xhat).abs() + u.abs())
    y = _act(u, act)
    tol_y = 1.1 * off_u + 8 * U * y.abs() + HALF[dtype] * y.abs() + 2.0 ** -130
    if dy is None:
        return tol_y
    slope = {"none": torch.ones_like(u), "relu": (u > 0).double(), "silu": torch.sigmoid(u) * (1 + u * (1 - torch.sigmoid(u)))}[act]
    du = dy * slope
    off_du = dy.abs() * (0.5 * off_u + 8 * U)
    if act == "relu":
        off_du = off_du + torch.where(u.abs() <= off_u, dy.abs(), 0.0)
    off_a = off_du.sum(1) + (d + 2) * U * du.abs().sum(1)                                        # [N, C]
    off_b = (off_du * xhat.abs() + du.abs() * off_x).sum(1) + (d + 4) * U * (du * xhat).abs().sum(1)
    tol_db = off_a.sum(0) + n * U * du.sum(1).abs().sum(0) + U * du.sum((0, 1)).abs()
    tol_dw = off_b.sum(0) + n * U * (du * xhat).sum(1).abs().sum(0) + U * (du * xhat).sum((0, 1)).abs()
    grp = lambda s: s.view(n, 1, groups, k).sum(3, keepdim=True) / (p * k)                       # noqa: E731
    a, bb = du.sum(1), (du * xhat).sum(1)
    m1, m2 = each(grp(a * w).expand(n, p, groups, k)), each(grp(bb * w).expand(n, p, groups, k))
    off_m1 = each(grp((off_a + (c + 4) * U * a.abs()) * w.abs())) + 4 * U * m1.abs()
    off_m2 = each(grp((off_b + (c + 4) * U * bb.abs()) * w.abs())) + 4 * U * m2.abs()
    r = each(rstd)
    size = (w * du).abs() + m1.abs() + (xhat * m2).abs()
    tol_dx = r * (w.abs() * off_du + off_m1 + xhat.abs() * off_m2 + off_x * m2.abs() + size * (each(off_r) + 6 * U))
    return tol_y, tol_dx + HALF[dtype] * (r * (w * du - m1 - xhat * m2)).abs() + 2.0 ** -130, tol_dw + 2.0 ** -130, tol_db + 2.0 ** -130


def _inputs(shape, dtype, seed, layout="channels_last", shift=0.5, spread=1.0):
    gen = torch.Generator().manual_seed(seed)
    n, c = shape[:2]
    per = (1, c) + (1,) * (len(shape) - 2)
    x = (spread * torch.randn(shape, generator=gen) * (0.5 + torch.rand(per, generator=gen)) + shift * torch.randn(per, generator=gen)).to(dtype)
    dy = torch.randn(shape, generator=gen).to(dtype)
    w, b = 1 + 0.3 * torch.randn(c, generator=gen), 0.3 * torch.randn(c, generator=gen)
    if layout == "channels_last":
        x, dy = (t.movedim(1, -1).contiguous().movedim(-1, 1) for t in (x, dy))
    return x.cuda(), w.cuda(), b.cuda(), dy.cuda()


def _flat(t):
    return t.detach().cpu().double().movedim(1, -1).reshape(t.shape[0], -1, t.shape[1])


def _check(x, w, b, dy, groups, act, eps=1e-5, affine=True):
    from erfnet_pytorch_amd.norm import group_norm_act
    x = x.detach().requires_grad_()
    w, b = (w.detach().requires_grad_(), b.detach().requires_grad_()) if affine else (None, None)
    y = group_norm_act(x, groups, w, b, eps, act)
    grads = torch.autograd.grad(y, (x, w, b) if affine else (x,), dy)
    assert y.dtype == x.dtype and y.shape == x.shape and y.movedim(1, -1).is_contiguous() and grads[0].shape == x.shape and grads[0].dtype == x.dtype
    with torch.no_grad():
        assert torch.equal(group_norm_act(x, groups, w, b, eps, act), y)
    c = x.shape[1]
    xd = _flat(x).requires_grad_()
    wd = (w.detach().cpu().double() if affine else torch.ones(c, dtype=torch.float64)).requires_grad_()
    bd = (b.detach().cpu().double() if affine else torch.zeros(c, dtype=torch.float64)).requires_grad_()
    yd = _ref(xd, wd, bd, groups, eps, act)
    want = torch.autograd.grad(yd, (xd, wd, bd), _flat(dy))
    tol = _tolerances(xd.detach(), wd.detach(), bd.detach(), _flat(dy), groups, eps, act, x.dtype)
    assert ((_flat(y) - yd.detach()).abs() <= tol[0]).all()
    assert ((_flat(grads[0]) - want[0]).abs() <= tol[1]).all()
    if affine:
        assert ((grads[1].cpu().double() - want[1]).abs() <= tol[2]).all() and ((grads[2].cpu().double() - want[2]).abs() <= tol[3]).all()


# channels that fill 16-byte chunks, that fill part of one, odd ones, more than a workgroup has threads; groups inside a chunk and over several
SHAPES = [((1, 16, 8, 16), 4), ((2, 128, 16, 32), 8), ((2, 128, 9, 7), 32), ((3, 30, 13, 11), 6), ((2, 27, 17, 5), 3), ((1, 64, 64, 64), 1),
          ((2, 20, 31, 33), 20), ((1, 2304, 3, 5), 9), ((2, 1030, 2, 3), 2), ((5, 8, 1, 1), 2), ((4, 6, 1, 2), 6), ((1, 1, 40, 50), 1),
          ((2, 4, 300, 301), 2), ((1, 16, 512, 256), 4), ((7, 32, 24), 4), ((9, 24), 3), ((1, 12, 3, 4, 5), 4), ((40, 16, 4, 8), 16)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", ["none", "relu", "silu"])
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_forward_and_gradients(shape, groups, act, dtype):
    _check(*_inputs(shape, dtype, 1), groups, act)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,groups", [((2, 128, 16, 32), 8), ((3, 30, 13, 11), 6), ((1, 64, 64, 64), 2)])
def test_means_far_from_zero_small_spreads_and_no_affine(shape, groups, dtype):
    for shift, spread, eps in ((300.0, 1.0, 1e-5), (0.0, 1e-4, 1e-5), (0.0, 1e4, 1e-3), (1.0, 1.0, 0.0)):
        x, w, b, dy = _inputs(shape, dtype, 2, shift=shift, spread=spread)
        _check(x, w, b, dy, groups, "silu", eps)
    _check(x, w, b, dy, groups, "relu", affine=False)


@pytest.mark.gpu
def test_one_outlier_does_not_cost_the_variance_its_digits():
    """The first value of a group 1e4 times the others' size: a shift by it would leave sums of squares that cancel."""
    x, w, b, dy = _inputs((2, 32, 64, 64), torch.float32, 3, shift=0.0)
    x[:, ::8, 0, 0] = 1e4
    _check(x, w, b, dy, 4, "none")


@pytest.mark.gpu
def test_constant_groups():
    """Variance 0: y = act(beta); the gradient is dy's own, centred, times 1 / sqrt(eps)."""
    x, w, b, dy = _inputs((2, 8, 8, 8), torch.float32, 4)
    x = torch.full_like(x, 0.75)
    _check(x, w, b, dy, 2, "silu")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_other_memory_layouts_and_types_of_parameters(dtype):
    """NCHW memory (copied), a slice of a larger map, an expanded gradient, bf16 parameters."""
    from erfnet_pytorch_amd.norm import group_norm_act
    x, w, b, dy = _inputs((2, 24, 10, 12), dtype, 5)
    want = group_norm_act(x, 4, w, b)
    assert torch.equal(group_norm_act(x.contiguous(), 4, w, b), want)
    big = torch.zeros(2, 10, 12, 30, dtype=dtype, device="cuda")
    big[..., 3:27] = x.permute(0, 2, 3, 1)
    assert torch.equal(group_norm_act(big[..., 3:27].permute(0, 3, 1, 2), 4, w, b), want)
    xr = x.clone().requires_grad_()
    d1, = torch.autograd.grad(group_norm_act(xr, 4, w, b), xr, torch.ones((), device="cuda", dtype=dtype).expand(x.shape))
    d2, = torch.autograd.grad(group_norm_act(xr, 4, w, b), xr, torch.ones_like(x))
    assert torch.equal(d1, d2)
    wb = w.bfloat16().requires_grad_()
    g, = torch.autograd.grad(group_norm_act(x, 4, wb, b).float().sum(), wb)
    assert g.dtype == torch.bfloat16 and torch.equal(group_norm_act(x, 4, wb.float(), b), group_norm_act(x, 4, wb, b))


@pytest.mark.gpu
def test_nan_and_infinity_stay_in_their_group():
    from erfnet_pytorch_amd.norm import group_norm_act
    x, w, b, dy = _inputs((3, 16, 8, 8), torch.float32, 6)
    clean = group_norm_act(x, 4, w, b)
    x[0, 5, 3, 3] = float("nan")
    x[1, 0, 0, 0] = float("inf")
    y = group_norm_act(x, 4, w, b)
    assert y[0, 4:8].isnan().all() and y[1, 0:4].isnan().any()
    keep = torch.ones_like(y, dtype=torch.bool)
    keep[0, 4:8] = False
    keep[1, 0:4] = False
    assert torch.equal(y[keep], clean[keep])


@pytest.mark.gpu
def test_gradient_against_differences():
    """Central differences of f = sum(r y) with h = 2^-5 along a random direction of length sqrt(size): three step sizes up to a factor
    of 2 must agree with the gradient to h^2 |f'''| / 6 + rounding; with x of spread 1 over 2 x 60 values and |r| <= 4, |f'''| <= 60 |r|_1
    / size per unit step is a wide bound, rounding 4000 U |r|_1 / h."""
    from erfnet_pytorch_amd.norm import group_norm_act
    x, w, b, r = _inputs((2, 6, 4, 5), torch.float32, 7)
    gen = torch.Generator().manual_seed(8)
    direction = torch.randn(x.shape, generator=gen).cuda()
    direction = direction / direction.abs().max()
    for act in ("none", "silu"):
        xr = x.clone().requires_grad_()
        g, = torch.autograd.grad(group_norm_act(xr, 2, w, b, 1e-5, act), xr, r)
        along = float((g.double() * direction.double()).sum())
        h = 2.0 ** -5
        f = [float((group_norm_act(x + s * h * direction, 2, w, b, 1e-5, act).double() * r.double()).sum()) for s in (1, -1)]
        size = float(r.double().abs().sum())
        assert abs((f[0] - f[1]) / (2 * h) - along) <= size * (h * h / 6 * 60 + 4000 * U / h)


@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups", [((1, 128, 16, 32), 8), ((2, 64, 64, 128), 8)])
def test_captured_calls_and_another_stream(shape, groups):
    from erfnet_pytorch_amd.norm import group_norm_act

    def both(x, w, b, dy):
        y = group_norm_act(x, groups, w, b, 1e-5, "silu")
        return [y.detach(), *torch.autograd.grad(y, (x, w, b), dy)]
    sets = []
    for i in range(2):
        x, w, b, dy = _inputs(shape, torch.bfloat16, 10 + i)
        sets.append((x.requires_grad_(), w.requires_grad_(), b.requires_grad_(), dy))
    both(*sets[0])
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, capture_error_mode="thread_local"):
            outs.append(both(*s))
        graphs.append(g)
    for rep in range(3):
        for i, s in enumerate(sets):
            with torch.no_grad():
                s[0].copy_(_inputs(shape, torch.bfloat16, 20 + 2 * rep + i)[0])
        for g in graphs:
            g.replay()
        want = [both(s[0].detach().clone().requires_grad_(), *s[1:]) for s in sets]
        torch.cuda.synchronize()
        for o, v in zip(outs, want):
            assert all(torch.equal(p, q) for p, q in zip(o, v))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = both(*sets[0])
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(there, want[0]))


@pytest.mark.gpu
def test_more_groups_than_one_launch_has_workgroups():
    """1.06 million groups: whole images from both sides of the 2^20th group against the formula."""
    from erfnet_pytorch_amd import train_ops as TO
    n, p, c = 1024, 600, 1040
    gen = torch.Generator(device="cuda").manual_seed(5)
    x, dy = (torch.randn(n, p, c, generator=gen, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    w, b = (torch.randn(c, generator=gen, device="cuda") for _ in range(2))
    y, stats = TO.group_norm_act_fwd(x, w, b, c, 1e-5, "silu")
    dx = TO.group_norm_act_bwd(dy, x, w, b, stats, c, "silu")[0]
    for i in (0, 2 ** 20 // c, 2 ** 20 // c + 1, n - 1):
        xd, wd, bd, dyd = x[i:i + 1].cpu().double().requires_grad_(), w.cpu().double(), b.cpu().double(), dy[i:i + 1].cpu().double()
        yd = _ref(xd, wd, bd, c, 1e-5, "silu")
        tol = _tolerances(xd.detach(), wd, bd, dyd, c, 1e-5, "silu", torch.bfloat16)
        assert ((y[i:i + 1].cpu().double() - yd.detach()).abs() <= tol[0]).all()
        assert ((dx[i:i + 1].cpu().double() - torch.autograd.grad(yd, xd, dyd)[0]).abs() <= tol[1]).all()


@pytest.mark.gpu
def test_offsets_that_pass_32_bits():
    """A map of 2^32 + 2^23 values whose pixels repeat with period 64: mean, variance and gradient means are those of one period.

    At most 4096 additions one after another (1024 workgroups share a map's pixels, two pixel lanes each: 2052 pixels a thread, and some
    tens to join them), d U = 2^-12.  In the forward pass 4 pixels are summed before they are joined: 2^-14 of the mean size 0.8 and of
    rstd, so off(u) <= 2^-14 (1 + |xhat|) <= 6 * 2^-14 for |xhat| <= 5, and y is off by 1.1 of that and half a step: 2^-10 + 2^-8 |y|.
    dx: |dy| off(u) / 2 <= 2^-10, the two means 2^-12 * 0.8 (1 + |xhat|) <= 2^-9, and half a step: 2^-8 + 2^-8 |dx|."""
    from erfnet_pytorch_amd import train_ops as TO
    n, p, c, groups = 8, 2 ** 19 + 2 ** 10, 1024, 8
    gen = torch.Generator().manual_seed(6)
    x, dy = (torch.randn(1, 64, c, generator=gen).bfloat16() for _ in range(2))
    big, dbig = (t.cuda().expand(n * p // 64, 64, c).reshape(n, p, c) for t in (x, dy))
    y, stats = TO.group_norm_act_fwd(big, None, None, groups, 1e-5, "silu")
    xd = x.double().requires_grad_()
    want = _ref(xd, torch.ones(c, dtype=torch.float64), torch.zeros(c, dtype=torch.float64), groups, 1e-5, "silu")
    dwant = torch.autograd.grad(want, xd, dy.double())[0]
    dx = TO.group_norm_act_bwd(dbig, big, None, None, stats, groups, "silu")[0]
    for i, at in ((0, 0), (n - 1, p - 64)):
        assert ((y[i, at:at + 64].cpu().double() - want.detach()[0]).abs() <= 2.0 ** -10 + 2.0 ** -8 * want.detach()[0].abs()).all()
        assert ((dx[i, at:at + 64].cpu().double() - dwant[0]).abs() <= 2.0 ** -8 * (1 + dwant[0].abs())).all()
        assert torch.equal(y[i, at:at + 64], y[0, :64]) and torch.equal(dx[i, at:at + 64], dx[0, :64])


@pytest.mark.gpu
def test_second_derivatives_are_refused():
    from erfnet_pytorch_amd.norm import group_norm_act
    x, w, b, dy = _inputs((1, 8, 4, 4), torch.float32, 12)
    y = group_norm_act(x.requires_grad_(), 2, w, b)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(y, x, dy, create_graph=True)


@pytest.mark.gpu
def test_module_and_empty_maps():
    from erfnet_pytorch_amd.norm import GroupNormAct2d, group_norm_act
    m = GroupNormAct2d(4, 16).cuda()
    ref = torch.nn.GroupNorm(4, 16)
    ref.load_state_dict(m.state_dict())
    x, _, _, dy = _inputs((2, 16, 8, 8), torch.float32, 9)
    assert torch.equal(m(x), group_norm_act(x, 4, m.weight, m.bias, 1e-5, "relu"))
    m(x).backward(dy)
    assert m.weight.grad.shape == (16,) and m.bias.grad.abs().sum() > 0
    for shape in ((0, 16, 4, 4), (2, 16, 0, 4)):
        e = torch.zeros(shape, device="cuda", requires_grad=True)
        m.zero_grad()
        y = m(e)
        y.sum().backward()
        assert y.shape == shape and (m.weight.grad == 0).all() and e.grad.shape == shape


# ------------------------------------------------------------------------------------------------ refusals (CPU)
def test_wrong_arguments_are_refused():
    from erfnet_pytorch_amd import train_ops
    from erfnet_pytorch_amd.norm import GroupNormAct2d, group_norm_act
    with pytest.raises(RuntimeError, match="MI355X"):
        group_norm_act(torch.zeros(1, 4, 2, 2), 2)
    with pytest.raises(ValueError, match="multiple"):
        GroupNormAct2d(3, 16)
    with pytest.raises(ValueError, match="activation"):
        GroupNormAct2d(4, 16, activation="gelu")
    f, x = train_ops.group_norm_act_fwd, torch.zeros(1, 2, 2, 4)
    with pytest.raises(TypeError):
        f(x.half(), None, None, 2, 1e-5, "relu")
    with pytest.raises(ValueError, match="groups"):
        f(x, None, None, 3, 1e-5, "relu")
    with pytest.raises(ValueError, match="groups"):
        f(x, None, None, 0, 1e-5, "relu")
    with pytest.raises(ValueError, match="activation"):
        f(x, None, None, 2, 1e-5, "tanh")
    with pytest.raises(ValueError, match="weight"):
        f(x, torch.zeros(5), None, 2, 1e-5, "relu")
    with pytest.raises(ValueError, match="bias"):
        f(x, None, torch.zeros(4, 1), 2, 1e-5, "relu")
    with pytest.raises(ValueError, match="eps"):
        f(x, None, None, 2, -1.0, "relu")
    with pytest.raises(ValueError, match="channels-last"):
        f(x.transpose(1, 3), None, None, 1, 1e-5, "relu")
    with pytest.raises(ValueError, match="on meta"):
        f(x, torch.zeros(4, device="meta"), None, 2, 1e-5, "relu")
    with pytest.raises(ValueError, match="dy"):
        train_ops.group_norm_act_bwd(x.bfloat16(), x, None, None, torch.zeros(2, 1, 2), 2, "relu")
    for bad in (torch.zeros(2, 1, 3), torch.zeros(2, 1, 2, dtype=torch.float64), torch.zeros(2, 1, 4)[..., ::2]):
        with pytest.raises(ValueError, match="stats"):
            train_ops.group_norm_act_bwd(x, x, None, None, bad, 2, "relu")


def test_abi_refuses_bad_arguments_without_a_gpu():
    from erfnet_pytorch_amd import _lib
    good = [16, 16, 0, 1, 6, 4, 2, 0, 0, 1e-5, 1, 16, 16, 16, 0]
    for i, bad in ((0, 0), (1, 0), (2, 2), (3, 0), (4, 0), (5, 0), (6, 0), (6, 3), (9, -1.0), (9, float("nan")), (10, 3), (10, -1), (11, 0), (12, 0), (13, 0)):
        args = list(good)
        args[i] = bad
        assert _lib.query("erf_group_norm_fwd", *args) == -1, i
    good = [16, 16, 16, 0, 1, 6, 4, 2, 0, 0, 1, 16, 16, 0, 0, 16, 0]
    for i, bad in ((0, 0), (1, 0), (2, 0), (3, 5), (4, 0), (5, 0), (6, 0), (7, 3), (10, 3), (11, 0), (12, 0), (15, 0)):
        args = list(good)
        args[i] = bad
        assert _lib.query("erf_group_norm_bwd", *args) == -1, i
    assert _lib.query("erf_group_norm_workspace_bytes", 0, 1, 6, 4, 3) == 0 and _lib.query("erf_group_norm_workspace_bytes", 0, 1, 6, 4, 2) > 0
