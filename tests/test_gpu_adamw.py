"""optim.AdamW (one launch over many tensors, moments in 32 or 8 bits) against the update formula in 64 bits.

Tolerances count roundings to nearest of 2^-24 relative (fp32) and 2^-8 (bf16):
  m = m b1 + g (1 - b1): the two constants and products round once each (4), the sum once, so the error is at most
  (2 + 1) 2^-24 (|m b1| + |g (1 - b1)|); 4 is used.  v: one product more, 5.
  The update u = step_size m / (sqrt(v) c + eps): m 3, sqrt(v) 4 / 2 + 1, c 1, product 1, sum 1, quotient 1, step_size 1 and the last
  product 1, relative to u's own size -- where m cancels, its error is relative to |m b1| + |g (1 - b1)| instead; 12 is used on that
  majorant.  p decay - u: constant, product, difference: 3 on |p| + |u|.
8-bit codes are rounded up or down: off by less than one step, 2^-3 relative or 2^-9 of the scale.
"""
import copy

import pytest
import torch

LR, BETAS, EPS, WD = 3e-3, (0.9, 0.999), 1e-8, 0.02
U = 2.0 ** -24


def _adamw(*a, **k):
    from erfnet_pytorch_amd.optim import AdamW
    return AdamW(*a, **k)


# ------------------------------------------------------------------------------------------------ refusals (CPU)
def test_constructor_refuses_what_it_cannot_do():
    p = torch.nn.Parameter(torch.zeros(4))
    for bad in (dict(state_bits=16), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(lr=-1.0), dict(lr=float("nan")), dict(eps=-1.0),
                dict(weight_decay=-1.0), dict(lr=torch.zeros(2))):
        with pytest.raises(ValueError):
            _adamw([p], **bad)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        _adamw([torch.nn.Parameter(torch.zeros(4, dtype=torch.float16))])
    with pytest.raises(ValueError, match="gaps or overlaps"):
        _adamw([torch.nn.Parameter(torch.zeros(4, 4)[:, ::2])])
    with pytest.raises(ValueError, match="gaps or overlaps"):
        _adamw([torch.nn.Parameter(torch.zeros(4, 1).expand(4, 4))])
    opt = _adamw([p])
    with pytest.raises(TypeError):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(2, dtype=torch.float64))]})
    assert len(opt.param_groups) == 1


def test_saved_settings_that_it_does_not_compute_are_refused_before_anything_is_loaded():
    p = torch.nn.Parameter(torch.zeros(3))
    opt = _adamw([p], lr=1e-2)
    for other in (torch.optim.AdamW([p], amsgrad=True), torch.optim.AdamW([p], maximize=True), torch.optim.Adam([p], weight_decay=0.1),
                  torch.optim.SGD([p], lr=0.1)):
        with pytest.raises(ValueError):
            opt.load_state_dict(other.state_dict())
        assert opt.param_groups[0]["lr"] == 1e-2
    bad = opt.state_dict()
    bad["param_groups"][0] = {**bad["param_groups"][0], "betas": (0.9, 1.0), "lr": 5.0}
    with pytest.raises(ValueError):
        opt.load_state_dict(bad)
    assert opt.param_groups[0]["lr"] == 1e-2
    for other in (torch.optim.AdamW([p], lr=0.5), torch.optim.Adam([p], lr=0.25)):              # Adam without weight decay is the same
        opt.load_state_dict(other.state_dict())
        assert opt.param_groups[0]["lr"] == other.param_groups[0]["lr"]


def test_cpu_parameters_are_refused_at_the_step_and_no_gradient_is_no_step():
    p = torch.nn.Parameter(torch.zeros(4))
    opt = _adamw([p])
    opt.step()
    p.grad = torch.ones(4)
    with pytest.raises(RuntimeError, match="MI355X"):
        opt.step()
    assert torch.equal(p.detach(), torch.zeros(4))


def test_the_watch_reports_what_changed():
    from erfnet_pytorch_amd.optim import _host
    ps = [torch.nn.Parameter(torch.zeros(2, 3)) for _ in range(3)]
    ps[0].grad, ps[2].grad = torch.zeros(2, 3), torch.zeros(2, 3)
    w = _host.ParamWatch()
    w.bind([ps[:1], ps[1:]])
    assert [w.look([ps[:1], ps[1:]]) for _ in range(2)] == [1, 0]
    old = ps[2].grad
    ps[2].grad = torch.zeros(2, 3)
    assert [w.look([ps]) for _ in range(2)] == [1, 0]
    ps[2].grad = old.t().contiguous().t()
    assert w.look([ps]) == 1 and w.copied() == [1] and w.look([ps]) == 1
    ps[2].grad = old
    assert w.look([ps]) == 1 and w.copied() == [] and w.look([ps]) == 0
    ps[0].data = torch.ones(2, 3)
    assert w.look([ps]) == 2 and w.look([ps[:2]]) == 2
    w.bind([ps])
    ps[1].grad = torch.zeros(2, 3)
    assert w.look([ps]) == 2
    before = ps[0]._version
    w.bump()
    assert ps[0]._version == before + 1
    with pytest.raises(ValueError, match="gradient"):
        ps[0].grad = torch.sparse_coo_tensor(torch.tensor([[0], [0]]), torch.tensor([1.0]), (2, 3))
        w.look([ps])


def test_the_watch_sees_other_shapes_at_the_same_place():
    """p.data replaced by a part or another order of itself: the tables describe something else then."""
    from erfnet_pytorch_amd.optim import _host
    for other in (lambda t: t[:2], lambda t: t.view(3, 4), lambda t: t.view(3, 4).t()):
        p = torch.nn.Parameter(torch.zeros(4, 3))
        p.grad = torch.zeros(4, 3)
        w = _host.ParamWatch()
        w.bind([[p]])
        assert [w.look([[p]]) for _ in range(2)] == [1, 0]
        p.grad = None
        p.data = other(p.data)
        p.grad = torch.zeros_like(p)
        assert w.look([[p]]) == 2


def test_parameters_put_into_a_group_by_hand_are_checked():
    p, h = torch.nn.Parameter(torch.zeros(4)), torch.nn.Parameter(torch.zeros(4, dtype=torch.float16))
    opt = _adamw([p])
    opt.param_groups[0]["params"].append(h)
    h.grad = torch.zeros_like(h)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        opt.step()


def test_parameters_that_share_memory_are_found():
    from erfnet_pytorch_amd.optim import _host
    t = torch.zeros(10)
    _host.adamw_no_overlap([t[:5], t[5:]])
    with pytest.raises(ValueError, match="share memory"):
        _host.adamw_no_overlap([t[5:], t[:6]])


def test_abi_refuses_bad_arguments_without_a_gpu():
    from erfnet_pytorch_amd import _lib
    good = [16, 16, 16, 1, 16, 0.9, 0.999, 1e-8, 0.0, 0, 32, 0, 0]
    for i, bad in ((0, 0), (1, 0), (2, 0), (3, 0), (4, 0), (5, 1.0), (6, -0.1), (7, -1.0), (9, 2), (10, 16)):
        args = list(good)
        args[i] = bad
        assert _lib.query("erf_adamw_step", *args) == -1, i
    assert _lib.query("erf_adamw_set_grads", 0, 16, 1, 0) == -1 and _lib.query("erf_adamw_set_grads", 16, 0, 1, 0) == -1
    assert _lib.query("erf_adamw_scale_block") == 256 and _lib.query("erf_adamw_chunk_elements") % 256 == 0


# ------------------------------------------------------------------------------------------------ the formula in 64 bits
def _reference(p, g, m, v, step, lr=LR, betas=BETAS, eps=EPS, wd=WD):
    """(new p, new m, new v, tolerances of the three) in float64."""
    p, g, m, v = (t.double() for t in (p, g, m, v))
    b1, b2 = betas
    size_m = (m * b1).abs() + (g * (1 - b1)).abs()
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g * g * (1 - b2)
    per = lr / (1 - b1 ** step) / (v.sqrt() / (1 - b2 ** step) ** 0.5 + eps)
    tiny = 2.0 ** -140                                    # below the smallest normal fp32 value rounding is absolute
    tol_u = 12 * U * per * size_m
    new = p * (1 - lr * wd) - per * m
    return new, m, v, tol_u + 3 * U * (p.abs() + (per * m).abs()) + tiny, 4 * U * size_m + tiny, 5 * U * v + tiny


SIZES = [1, 3, 4, 255, 256, 257, 1023, 4095, 4096, 4097, 12345]


def _tensors(sizes, dtype, seed, offset=0):
    gen = torch.Generator().manual_seed(seed)
    out = []
    for n in sizes:
        t = [torch.randn(n + offset, generator=gen) * s for s in (0.1, 1e-2)]
        out.append([a.to(dtype).cuda()[offset:] for a in t])
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [0, 1])
def test_32_bit_states_against_the_formula_over_steps(dtype, offset):
    ts = _tensors(SIZES, dtype, 1, offset)
    params = [torch.nn.Parameter(p) for p, _ in ts]
    opt = _adamw(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=WD)
    m = [torch.zeros(n, device="cuda") for n in SIZES]
    v = [torch.zeros(n, device="cuda") for n in SIZES]
    gen = torch.Generator(device="cuda").manual_seed(5)
    for step in (1, 2, 3):
        before = [p.detach().clone() for p in params]
        for p in params:
            p.grad = (1e-2 * torch.randn(p.shape, device="cuda", generator=gen)).to(dtype)
        opt.step()
        for i, p in enumerate(params):
            rp, rm, rv, tp, tm, tv = _reference(before[i], p.grad, m[i], v[i], step)
            m[i], v[i] = opt.state[p]["exp_avg"].clone(), opt.state[p]["exp_avg_sq"].clone()
            if dtype == torch.bfloat16:
                tp = tp + 2.0 ** -8 * rp.abs()
            assert ((p.double() - rp).abs() <= tp).all() and ((m[i].double() - rm).abs() <= tm).all() and ((v[i].double() - rv).abs() <= tv).all(), SIZES[i]
    assert all(float(s["step"]) == 3 for s in opt.state_dict()["state"].values())


def _decoded(opt, p, key):
    st = opt.state[p]
    return st[key].float().reshape(-1).double() * st[key + "_scale"].double().repeat_interleave(256)[:p.numel()]


def _check_codes(opt, p, key, want, tol):
    """Codes within one step of `want` (plus want's own tolerance), scales the right power of two, 0 only where nothing is left."""
    scale = opt.state[p][key + "_scale"].double()
    each = scale.repeat_interleave(256)[:p.numel()]
    got = _decoded(opt, p, key)
    step = torch.maximum(want.abs() * 2.0 ** -3, each * 2.0 ** -9)
    assert ((got - want).abs() <= step + tol).all()
    assert torch.equal(torch.frexp(scale)[0], torch.full_like(scale, 0.5))
    n = p.numel()
    most = torch.stack([want[i:i + 256].abs().max() for i in range(0, n, 256)])
    live = most > 2.0 ** -100
    ratio = (most / scale)[live]
    assert ((ratio <= 448 * (1 + 1e-5)) & (ratio >= 224 * (1 - 1e-5))).all()
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [0, 1])
def test_8_bit_states_against_the_formula_over_steps(dtype, offset):
    ts = _tensors(SIZES, dtype, 2, offset)
    params = [torch.nn.Parameter(p) for p, _ in ts]
    opt = _adamw(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=WD, state_bits=8, seed=7)
    gen = torch.Generator(device="cuda").manual_seed(6)
    m = [torch.zeros(n, device="cuda") for n in SIZES]
    v = [torch.zeros(n, device="cuda") for n in SIZES]
    for step in (1, 2, 3, 4):
        before = [p.detach().clone() for p in params]
        for p in params:
            spread = torch.exp(4 * torch.randn(p.shape, device="cuda", generator=gen))
            p.grad = (1e-3 * spread * torch.randn(p.shape, device="cuda", generator=gen)).to(dtype)
            p.grad[::5] = 0
        opt.step()
        for i, p in enumerate(params):
            rp, rm, rv, tp, tm, tv = _reference(before[i], p.grad, m[i], v[i], step)
            if dtype == torch.bfloat16:
                tp = tp + 2.0 ** -8 * rp.abs()
            assert ((p.double() - rp).abs() <= tp).all(), SIZES[i]
            gm = _check_codes(opt, p, "exp_avg", rm, tm)
            gr = _check_codes(opt, p, "exp_avg_sq_root", rv.sqrt(), 4 * U * rv.sqrt())
            assert ((gr > 0) == (rv.float() > 0)).all()             # sqrt(v) is 0 only where v is
            m[i], v[i] = gm.float(), gr.float().square()


@pytest.mark.gpu
def test_8_bit_rounding_is_fair_and_lets_v_fall():
    """With constant gradients of one size the mean of the decoded states is the state: the rounding of n elements has a variance of
    at most step^2 / 4 each, so the mean is within 6 * step / 2 / sqrt(n) (the 16 random bits add 2^-16 of a step).  With gradient 0
    a v of 32 bits falls by b2 a step; sqrt(v) rounded to nearest would stay where it is for ever."""
    n = 1 << 16
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    opt = _adamw([p], lr=0.0, betas=BETAS, eps=EPS, weight_decay=0.0, state_bits=8, seed=3)
    p.grad = torch.full((n,), 0.37, device="cuda")
    opt.step()
    m1, r1 = (1 - BETAS[0]) * 0.37, ((1 - BETAS[1]) * 0.37 ** 2) ** 0.5
    fair = 6 / 2 / n ** 0.5 + 2.0 ** -16
    for key, want in (("exp_avg", m1), ("exp_avg_sq_root", r1)):
        got = _decoded(opt, p, key)
        assert abs(float(got.mean()) - want) <= want * 2.0 ** -3 * fair and got.unique().numel() <= 2
    # many steps without a gradient: the mean of sqrt(v) follows b2^(t / 2) sqrt(v).  Each step's rounding adds a variance of at most
    # step^2 / 4 per element to what the steps before left; it shrinks with the rest
    p.grad = torch.zeros(n, device="cuda")
    steps = 400
    for _ in range(steps):
        opt.step()
    want = r1 * BETAS[1] ** (steps / 2)
    assert abs(float(_decoded(opt, p, "exp_avg_sq_root").mean()) - want) <= r1 * 2.0 ** -3 * fair * (steps + 1) ** 0.5 + 2.0 ** -9 * want
    # the momentum is below 1e-19 of its start by now; where it rounds to 0 it stays there
    assert float(_decoded(opt, p, "exp_avg").abs().max()) <= m1 * 1e-3


@pytest.mark.gpu
def test_the_same_run_gives_the_same_bits_and_another_seed_others():
    def run(seed):
        (p, _), = _tensors([5000], torch.float32, 3)
        p = torch.nn.Parameter(p)
        opt = _adamw([p], lr=LR, state_bits=8, seed=seed)
        for k in range(3):
            p.grad = torch.sin(torch.arange(5000, device="cuda") * (k + 1.0))
            opt.step()
        return p.detach().clone(), opt.state[p]["exp_avg"].view(torch.uint8).clone()
    a, b, c = run(1), run(1), run(2)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and not torch.equal(a[1], c[1])


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_values_that_are_not_finite_stay_where_they_are(bits):
    n = 600
    p = torch.nn.Parameter(torch.ones(n, device="cuda"))
    opt = _adamw([p], lr=LR, state_bits=bits)
    g = torch.full((n,), 0.01, device="cuda")
    g[5], g[300], g[301] = float("nan"), float("inf"), -float("inf")
    p.grad = g
    opt.step()
    p.grad = torch.full((n,), 0.01, device="cuda")
    opt.step()
    bad = torch.zeros(n, dtype=torch.bool, device="cuda")
    bad[5] = bad[300] = bad[301] = True
    assert torch.equal(torch.isnan(p.detach()), bad)
    q = torch.nn.Parameter(torch.ones(n, device="cuda"))
    clean = _adamw([q], lr=LR, state_bits=bits)
    for _ in range(2):
        q.grad = torch.full((n,), 0.01, device="cuda")
        clean.step()
    assert torch.equal(p.detach()[~bad], q.detach()[~bad])


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_nothing_beside_the_tensors_is_written(bits):
    arena, garena = torch.full((3000,), 7.0, device="cuda"), torch.full((3000,), 9.0, device="cuda")
    spans = [(3, 1), (10, 257), (301, 1000), (1501, 255)]
    params = []
    for a, n in spans:
        p = torch.nn.Parameter(arena[a:a + n])
        p.grad = garena[a:a + n]
        params.append(p)
    opt = _adamw(params, lr=LR, state_bits=bits)
    codes = torch.full((2, 3000), 0x11, dtype=torch.uint8, device="cuda")
    scales = torch.full((2, 64), 5.0, device="cuda")
    if bits == 8:
        at = 0
        for p, (a, n) in zip(params, spans):
            k = -(-n // 256)
            codes[:, a:a + n] = 0
            opt.state[p] = {"step": torch.zeros(()), "exp_avg": codes[0, a:a + n].view(torch.float8_e4m3fn), "exp_avg_scale": scales[0, at:at + k],
                            "exp_avg_sq_root": codes[1, a:a + n].view(torch.float8_e4m3fn), "exp_avg_sq_root_scale": scales[1, at:at + k]}
            at += k + 1
    opt.step()
    inside = torch.zeros(3000, dtype=torch.bool, device="cuda")
    for a, n in spans:
        inside[a:a + n] = True
    assert (arena[~inside] == 7.0).all() and (arena[inside] != 7.0).all() and (garena == 9.0).all()
    if bits == 8:
        assert (codes[:, ~inside] == 0x11).all() and (codes[:, inside] != 0x11).any()
        at = 0
        for _, n in spans:
            k = -(-n // 256)
            assert (scales[:, at:at + k] != 5.0).all() and (scales[:, at + k] == 5.0).all()
            at += k + 1


@pytest.mark.gpu
def test_a_tensor_of_more_than_2_to_the_32_elements():
    """Its last elements get the bits that a small tensor of the same values gets."""
    n, tail = 2 ** 32 + 5000, 9000
    gen = torch.Generator().manual_seed(9)
    end, grad = (torch.randn(tail, generator=gen).bfloat16().cuda() for _ in range(2))
    p, q = torch.nn.Parameter(torch.zeros(n, dtype=torch.bfloat16, device="cuda")), torch.nn.Parameter(end.clone())
    p.data[-tail:] = end
    p.grad, q.grad = torch.zeros_like(p), grad
    p.grad[-tail:] = grad
    opt = _adamw([p, q], lr=1e-2)
    opt.step()
    assert torch.equal(p.detach()[-tail:], q.detach()) and float(p.detach()[:-tail].abs().max()) == 0.0
    for k in ("exp_avg", "exp_avg_sq"):
        assert torch.equal(opt.state[p][k][-tail:], opt.state[q][k])


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_groups_missing_gradients_and_layouts(bits):
    """Groups with settings of their own, parameters without a gradient (left alone, with their own step count), channels-last
    parameters, gradients of other strides than their parameter's, empty parameters: as one optimizer per parameter."""
    def make():
        gen = torch.Generator().manual_seed(11)
        ps = [torch.randn(8, 4, 3, 3, generator=gen).cuda().contiguous(memory_format=torch.channels_last), torch.randn(700, generator=gen).cuda(),
              torch.randn(0, 5, generator=gen).cuda(), torch.randn(33, 65, generator=gen).cuda().t(), torch.randn(300, generator=gen).cuda().bfloat16()]
        return [torch.nn.Parameter(p) for p in ps]

    def grads(ps, k):
        gen = torch.Generator().manual_seed(100 + k)
        for i, p in enumerate(ps):
            g = torch.randn(p.shape, generator=gen).to(p.dtype).cuda()
            p.grad = None if (i == 1 and k == 1) else g
    a, b = make(), make()
    opt = _adamw([{"params": a[:2], "lr": 1e-2}, {"params": a[2:], "weight_decay": 0.3}], lr=LR, state_bits=bits, seed=9)
    for k in range(4):
        grads(a, k)
        opt.step()
    sd = opt.state_dict()["state"]
    assert [float(sd[i]["step"]) for i in (0, 1, 3, 4)] == [4, 3, 4, 4] and 2 not in sd
    for i, p in enumerate(b):
        if bits == 8 and i > 0:
            continue                                  # the random bits go by the position among all parameters: only the first one's are alike
        one = _adamw([p], lr=1e-2 if i < 2 else LR, weight_decay=1e-2 if i < 2 else 0.3, state_bits=bits, seed=9)
        for k in range(4):
            grads(b, k)
            one.step()
        assert torch.equal(a[i].detach(), p.detach()), i


@pytest.mark.gpu
def test_wrong_gradients_and_states_are_refused():
    p = torch.nn.Parameter(torch.zeros(300, device="cuda"))
    p.grad = torch.sparse_coo_tensor(torch.tensor([[1]]), torch.tensor([1.0]), (300,)).cuda()
    with pytest.raises(ValueError, match="gradient"):
        _adamw([p]).step()
    p.grad = torch.ones(300, device="cuda")
    for bits, name in ((32, "exp_avg_sq"), (8, "exp_avg"), (8, "exp_avg_scale")):
        opt = _adamw([p], state_bits=bits)
        opt.step()
        opt.state[p][name] = torch.zeros(7, device="cuda")
        opt.refresh()
        with pytest.raises(ValueError, match="state"):
            opt.step()
    with pytest.raises(ValueError, match="share memory"):
        q = torch.nn.Parameter(p.data[10:])
        q.grad = torch.ones(290, device="cuda")
        _adamw([p, q]).step()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_saved_and_loaded_states_go_on_as_if_nothing_had_happened(bits, tmp_path):
    def make():
        return [torch.nn.Parameter(p) for p, _ in _tensors([300, 5000], torch.float32, 21)] + \
               [torch.nn.Parameter(p) for p, _ in _tensors([777], torch.bfloat16, 22)]

    def grads(ps, k):
        for i, p in enumerate(ps):
            p.grad = torch.cos(torch.arange(p.numel(), device="cuda") * (k + 1.5) + i).to(p.dtype)
    a = make()
    opt = _adamw(a, lr=LR, state_bits=bits)
    for k in range(3):
        grads(a, k)
        opt.step()
    torch.save(opt.state_dict(), tmp_path / "opt.pt")
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    other = _adamw(b, lr=1.0, state_bits=bits)
    other.load_state_dict(torch.load(tmp_path / "opt.pt", weights_only=True))
    third = copy.deepcopy(opt)
    c = [p for g in third.param_groups for p in g["params"]]
    for k in (3, 4):
        for ps, o in ((a, opt), (b, other), (c, third)):
            grads(ps, k)
            o.step()
    for x, y, z in zip(a, b, c):
        assert torch.equal(x.detach(), y.detach()) and torch.equal(x.detach(), z.detach())
    assert all(float(s["step"]) == 5 for s in other.state_dict()["state"].values())


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("lr_tensor", [False, True])
def test_captured_steps_count_and_follow_the_learning_rate(bits, lr_tensor):
    """Replays of a captured step (with its gradients in static memory, eager steps and other gradients between) give the bits of
    the launched steps."""
    def run(graphed):
        ps = [torch.nn.Parameter(p) for p, _ in _tensors([300, 9000], torch.float32, 31)]
        lr = torch.full((1,), 1e-3, dtype=torch.float64, device="cuda") if lr_tensor else 1e-3
        opt = _adamw(ps, lr=lr, state_bits=bits)
        static = [torch.zeros_like(p) for p in ps]

        def fill(k):
            for i, s in enumerate(static):
                s.copy_(torch.cos(torch.arange(s.numel(), device="cuda") * (k + 0.5) + i))
            for p, s in zip(ps, static):
                p.grad = s

        def set_lr(v):
            if lr_tensor:
                lr.fill_(v)
            else:
                opt.param_groups[0]["lr"] = v
        fill(0)
        opt.step()
        graph = torch.cuda.CUDAGraph()
        if graphed:
            torch.cuda.synchronize()
            with torch.cuda.graph(graph, capture_error_mode="thread_local"):
                opt.step()

        def go(k):
            fill(k)
            if graphed:
                opt.refresh_lr()
                graph.replay()
                opt.note_replay()
            else:
                opt.step()
        go(1)
        go(2)
        for p in ps:                                   # an eager step with gradients elsewhere, between two replays
            p.grad = torch.full_like(p, 0.25)
        opt.step()
        set_lr(5e-3)
        go(3)
        torch.cuda.synchronize()
        go(4)
        return [p.detach().clone() for p in ps], [float(s["step"]) for s in opt.state_dict()["state"].values()]
    (a, ca), (b, cb) = run(False), run(True)
    assert ca == cb == [6.0, 6.0] and all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.gpu
def test_hooks_schedulers_and_closures():
    p = torch.nn.Parameter(torch.ones(300, device="cuda"))
    opt = _adamw([p], lr=0.5, weight_decay=0.0, betas=(0.0, 0.0), eps=0.0)
    sched = torch.optim.lr_scheduler.StepLR(opt, 1, 0.5)
    seen = []
    handles = [opt.register_step_pre_hook(lambda o, a, k: seen.append("pre")), opt.register_step_post_hook(lambda o, a, k: seen.append("post"))]

    def closure():
        p.grad = torch.full_like(p, 3.0)
        return 7.0
    assert opt.step(closure) == 7.0 and seen == ["pre", "post"] and torch.equal(p.detach(), torch.full_like(p, 0.5))
    sched.step()
    for h in handles:
        h.remove()
    opt.step()
    assert seen == ["pre", "post"] and torch.equal(p.detach(), torch.full_like(p, 0.25))


@pytest.mark.gpu
def test_the_optimizer_keeps_no_gradient_alive():
    import weakref
    p = torch.nn.Parameter(torch.ones(1000, device="cuda"))
    opt = _adamw([p])
    p.grad = torch.ones_like(p)
    gone = weakref.ref(p.grad)
    opt.step()
    opt.zero_grad(set_to_none=True)
    assert gone() is None


@pytest.mark.gpu
def test_capture_before_the_first_step_and_a_changed_rate_inside_a_capture_are_refused():
    p = torch.nn.Parameter(torch.zeros(10, device="cuda"))
    p.grad = torch.ones(10, device="cuda")
    opt = _adamw([p])
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), capture_error_mode="thread_local"):
            opt.step()
    opt.step()
    opt.param_groups[0]["lr"] = 0.5
    with pytest.raises(RuntimeError, match="refresh_lr"):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), capture_error_mode="thread_local"):
            opt.step()
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_gradients_made_inside_the_capture_and_another_stream():
    """zero_grad(set_to_none=True), forward, backward and step in one graph; and steps issued on a side stream."""
    w0 = torch.randn(64, 64, generator=torch.Generator().manual_seed(1)).cuda()
    x = torch.randn(64, 64, generator=torch.Generator().manual_seed(2)).cuda()

    def one(p, opt):
        opt.zero_grad(set_to_none=True)
        p.grad, = torch.autograd.grad((x * p).square(), p, torch.ones_like(x))
        opt.step()
    p, q = torch.nn.Parameter(w0.clone()), torch.nn.Parameter(w0.clone())
    po, qo = _adamw([p], lr=1e-2), _adamw([q], lr=1e-2)
    one(p, po)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one(q, qo)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, capture_error_mode="thread_local"):
        one(p, po)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        one(q, qo)
        assert torch.equal(p.detach(), q.detach())


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_replays_between_steps_with_other_gradients_count_on(bits):
    """Eager steps without one of the captured step's gradients, without any, and with one more, between its replays: the bits and the
    counts of launched steps."""
    def run(graphed):
        ps = [torch.nn.Parameter(p) for p, _ in _tensors([300, 9000, 77], torch.float32, 41)]
        opt = _adamw(ps, lr=1e-3, state_bits=bits)
        static = [torch.zeros_like(p) for p in ps]

        def fill(k, which):
            for i, (p, s) in enumerate(zip(ps, static)):
                s.copy_(torch.cos(torch.arange(s.numel(), device="cuda") * (k + 0.5) + i))
                p.grad = s if i in which else None
        fill(0, (0, 1))
        opt.step()
        graph = torch.cuda.CUDAGraph()
        if graphed:
            torch.cuda.synchronize()
            with torch.cuda.graph(graph, capture_error_mode="thread_local"):
                opt.step()

        def go(k):
            fill(k, (0, 1))
            if graphed:
                graph.replay()
                opt.note_replay()
            else:
                opt.step()
            torch.cuda.synchronize()
        go(1)
        for k, which in enumerate(((0,), (), (1,), (0, 2), (2,), (0, 1, 2))):
            fill(10 + k, which)
            opt.step()
            go(20 + 2 * k)
            go(21 + 2 * k)
        return [p.detach().clone() for p in ps], [float(s["step"]) for s in opt.state_dict()["state"].values()], \
            [v for p in ps for k, v in opt.state[p].items() if k != "step"]
    (a, ca, sa), (b, cb, sb) = run(False), run(True)
    assert ca == cb == [17.0, 16.0, 3.0] and all(torch.equal(x, y) for x, y in zip(a, b))
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(sa, sb))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_tensor_without_a_gradient_is_left_alone(bits):
    """Its address in the table is NULL: values, moments and count stay, and it goes on where it was."""
    ps = [torch.nn.Parameter(p) for p, _ in _tensors([5000, 5000], torch.float32, 51)]
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    opt, other = _adamw(ps, lr=LR, state_bits=bits), _adamw(qs[:1], lr=LR, state_bits=bits)

    def mine():
        return [ps[0].detach()] + [v for k, v in opt.state[ps[0]].items() if k != "step"]
    for k in range(4):
        g = torch.cos(torch.arange(5000, device="cuda") * (k + 1.5))
        ps[0].grad, ps[1].grad = (g if k != 2 else None), g
        if k == 2:
            before = [t.clone() for t in mine()]
        opt.step()
        if k == 2:
            assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(before, mine()))
            continue
        qs[0].grad = g
        other.step()
    assert torch.equal(ps[0].detach(), qs[0].detach())
    assert [float(opt.state_dict()["state"][i]["step"]) for i in (0, 1)] == [3, 4]


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("eps", [0.0, 1e-45, 1e-39, 2.0 ** -126, 1e-8, 1.0, 1e30, 1e38, 1e300])
def test_every_size_of_eps(bits, eps):
    """Elements whose moments are 0 (their update is 0 / eps) only decay; the others follow the formula with eps as the fp32 value that
    the kernel has.  With eps = 0 an element without moments has no update: 0 / 0."""
    gen = torch.Generator().manual_seed(61)
    start = torch.randn(5000, generator=gen).cuda()
    g = (1e-2 * torch.randn(5000, generator=gen)).cuda()
    g[::3] = 0
    p = torch.nn.Parameter(start.clone())
    opt = _adamw([p], lr=LR, betas=BETAS, eps=eps, weight_decay=WD, state_bits=bits)
    p.grad = g
    opt.step()
    zero = torch.zeros(5000, device="cuda")
    rp, _, _, tp, _, _ = _reference(start, g, zero, zero, 1, eps=float(torch.tensor(eps, dtype=torch.float64).float()))
    if eps == 0.0:
        assert torch.equal(torch.isnan(p.detach()), g == 0)
        rp, tp = rp[g != 0], tp[g != 0]
        assert ((p.detach()[g != 0].double() - rp).abs() <= tp).all()
        return
    assert ((p.detach().double() - rp).abs() <= tp).all()


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-17, 2e-18, 1e-18, 1e-19, 1e-20])
def test_8_bit_moments_of_tiny_gradients(size):
    """v = (1 - b2) g^2 is subnormal below |g| of about 3e-18, a multiple of 2^-149: sqrt(v) is that of the v that fp32 holds, to a
    half step (U), and its code is off by less than a step.  Gradients of ordinary size beside them, in another scale block, and
    among them, where the tiny ones' codes are the smallest."""
    p = torch.nn.Parameter(torch.zeros(768, device="cuda"))
    opt = _adamw([p], lr=LR, betas=BETAS, eps=EPS, weight_decay=0.0, state_bits=8)
    g = size * (1 + torch.arange(768, device="cuda") / 768)
    g[256:512] = 0.5
    g[600] = 0.25
    p.grad = g
    opt.step()
    omb2 = torch.tensor(1 - BETAS[1], dtype=torch.float64).float().cuda()
    v = g * g * omb2                                          # as the kernel rounds them
    want = v.double().sqrt()
    got = _decoded(opt, p, "exp_avg_sq_root")
    each = opt.state[p]["exp_avg_sq_root_scale"].double().repeat_interleave(256)
    assert ((got - want).abs() <= torch.maximum(want * 2.0 ** -3, each * 2.0 ** -9) * (1 + 1e-6) + U * want).all()
    assert ((got > 0) == (v > 0)).all()
    first = want[:256].max()
    if float(first) > 0:
        assert 224 * (1 - 1e-5) <= float(first / each[0]) <= 448 * (1 + 1e-5)
