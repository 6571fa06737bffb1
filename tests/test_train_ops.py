"""Group norm, label log probabilities and AdamW together: as registered ops (schema, fake kernels, no CPU kernel) and as the pieces
of one training step."""
import math

import pytest
import torch

from erfnet_pytorch_amd import train_ops as TO

T = torch.ops.erfnet_mi355
U = 2.0 ** -24


def _samples(dev, dtype=torch.bfloat16):
    """op name -> [(args, expected outputs (shape, dtype, strides or None))]"""
    def t(*shape, dt=dtype):
        return torch.empty(shape, dtype=dt, device=dev)
    f, i = torch.float32, torch.int64
    maps, rows, last = t(2, 20, 8, 16), t(6, 1000), t(2, 20, 8, 16).contiguous(memory_format=torch.channels_last)
    x = t(2, 8, 16, 24)

    def fwd(z, k, target=True):
        pos = (z.shape[0], *z.shape[2:])
        tgt = t(*pos, dt=i) if target else None
        top = (pos[0], k, *pos[1:])
        return (z, tgt, k, -100), [(pos if target else (0,), f), (pos, f), ((2, *pos), f), (top, f), (top, i)]

    def bwd(z, k):
        pos = (z.shape[0], *z.shape[2:])
        top = (pos[0], k, *pos[1:])
        return (z, t(*pos, dt=i), t(2, *pos, dt=f), t(*pos, dt=f), t(*top, dt=i), t(*pos, dt=f), t(*pos, dt=f), t(*top, dt=f) if k else None, -100), [(tuple(z.shape), dtype)]
    return {
        "class_log_probs_fwd": [fwd(maps, 3), fwd(rows, 5), fwd(last, 2), fwd(maps, 0, False)],
        "class_log_probs_bwd": [bwd(maps, 3), bwd(rows, 0), bwd(last, 2)],
        "group_norm_act_fwd": [((x, t(24, dt=f), t(24, dt=f), 4, 1e-5, "relu"), [((2, 8, 16, 24), dtype), ((2, 2, 4), f)]),
                               ((x, None, None, 24, 1e-5, "silu"), [((2, 8, 16, 24), dtype), ((2, 2, 24), f)])],
        "group_norm_act_bwd": [((x, x, t(24, dt=f), None, t(2, 2, 4, dt=f), 4, "none"), [((2, 8, 16, 24), dtype), ((24,), f), ((24,), f)])],
    }


def _one_pixel(dev):
    """The same for maps of one pixel."""
    def t(*shape, dt=torch.float32):
        return torch.empty(shape, dtype=dt, device=dev)
    f, i, z = torch.float32, torch.int64, t(6, 20, 1, 1)
    return {"class_log_probs_fwd": [((z, None, 3, -100), [((0,), f), ((6, 1, 1), f), ((2, 6, 1, 1), f), ((6, 3, 1, 1), f), ((6, 3, 1, 1), i)])],
            "class_log_probs_bwd": [((z, t(6, 1, 1, dt=i), t(2, 6, 1, 1), t(6, 1, 1), t(6, 0, 1, 1, dt=i), t(6, 1, 1), None, None, -100), [((6, 20, 1, 1), f)])]}


def _outs(res):
    return list(res) if isinstance(res, (tuple, list)) else [res]


def test_every_op_is_registered_with_a_schema_a_device_kernel_and_a_fake_kernel():
    assert set(TO.OPS) == set(_samples("meta"))
    for name in TO.OPS:
        op = getattr(T, name).default
        assert op._schema.name == f"erfnet_mi355::{name}"
        assert torch._C._dispatch_has_kernel_for_dispatch_key(op.name(), "CUDA") and torch._C._dispatch_has_kernel_for_dispatch_key(op.name(), "Meta")
        assert not torch._C._dispatch_has_kernel_for_dispatch_key(op.name(), "CPU"), name


@pytest.mark.parametrize("name", sorted(_samples("meta")))
def test_fake_kernels_give_shapes_on_meta_tensors(name):
    for args, want in _samples("meta")[name]:
        got = _outs(getattr(T, name)(*args))
        assert [(tuple(o.shape), o.dtype) for o in got] == want and all(o.device.type == "meta" for o in got)


def test_ops_trace_under_fake_tensor_mode():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(4, 64, 128, 64, dtype=torch.bfloat16, device="cuda")
        y, stats = T.group_norm_act_fwd(x, torch.empty(64, device="cuda"), None, 8, 1e-5, "silu")
        z = torch.empty(4, 20, 64, 128, device="cuda").contiguous(memory_format=torch.channels_last)
        lp, ent, st, top, idx = T.class_log_probs_fwd(z, torch.empty(4, 64, 128, dtype=torch.int64, device="cuda"), 3, -100)
        dz = T.class_log_probs_bwd(z, torch.empty(4, 64, 128, dtype=torch.int64, device="cuda"), st, ent, idx, lp, ent, top, -100)
    assert tuple(y.shape) == (4, 64, 128, 64) and y.device.type == "cuda" and tuple(stats.shape) == (2, 4, 8)
    assert tuple(top.shape) == (4, 3, 64, 128) and top.stride() == idx.stride() == (64 * 128 * 3, 1, 128 * 3, 3)
    assert dz.is_contiguous(memory_format=torch.channels_last)


@pytest.mark.parametrize("name", sorted(_samples("meta")))
def test_ops_trace_with_dynamic_shapes(name):
    """Sizes as symbols: shapes, types and strides of the fixed sizes they stand for."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.symbolic_shapes import DimDynamic, ShapeEnv, StatelessSymbolicContext
    op = getattr(T, name)
    samples = list(_samples("meta")[name])
    if name.startswith("class_log_probs"):                  # one pixel a map: rows, whatever the strides
        samples += [s for s in _one_pixel("meta")[name]]
    for args, want in samples:
        fixed = _outs(op(*args))
        mode = FakeTensorMode(shape_env=ShapeEnv())

        def symbols(t):
            if not isinstance(t, torch.Tensor):
                return t
            return mode.from_tensor(t, symbolic_context=StatelessSymbolicContext(dynamic_sizes=[DimDynamic.DYNAMIC] * t.dim()))
        args = [symbols(a) for a in args]
        with mode:
            got = _outs(op(*args))
        assert any(isinstance(n, torch.SymInt) for o in got for n in o.shape)
        assert [(tuple(int(n) for n in o.shape), o.dtype) for o in got] == want
        for o, f in zip(got, fixed):
            assert all(int(a) == b for a, b, n in zip(o.stride(), f.stride(), f.shape) if n > 1)


def test_dynamic_shapes_that_do_not_fit_are_refused():
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.symbolic_shapes import DimDynamic, ShapeEnv, StatelessSymbolicContext
    mode = FakeTensorMode(shape_env=ShapeEnv())

    def symbols(*shape, dtype=torch.float32):
        t = torch.empty(shape, dtype=dtype, device="meta")
        return mode.from_tensor(t, symbolic_context=StatelessSymbolicContext(dynamic_sizes=[DimDynamic.DYNAMIC] * t.dim()))
    x, z = symbols(2, 8, 16, 24), symbols(4, 30, 5)
    with mode:
        for call in (lambda: T.group_norm_act_fwd(x, None, None, 5, 1e-5, "relu"), lambda: T.group_norm_act_fwd(x, None, None, 4, 1e-5, "gelu"),
                     lambda: T.group_norm_act_fwd(x, symbols(25), None, 4, 1e-5, "relu"), lambda: T.group_norm_act_fwd(x.transpose(1, 2), None, None, 4, 1e-5, "relu"),
                     lambda: T.group_norm_act_bwd(symbols(2, 8, 16, 12), x, None, None, symbols(2, 2, 4), 4, "relu"),
                     lambda: T.class_log_probs_fwd(z, None, 31, -100), lambda: T.class_log_probs_fwd(z, symbols(4, 6, dtype=torch.int64), 0, -100)):
            with pytest.raises(ValueError):
                call()
        with pytest.raises(TypeError):
            T.class_log_probs_fwd(symbols(4, 30, dtype=torch.float16), None, 0, -100)


def test_cpu_tensors_are_refused():
    with pytest.raises(NotImplementedError):
        T.group_norm_act_fwd(torch.zeros(1, 2, 2, 4), None, None, 2, 1e-5, "relu")
    with pytest.raises(NotImplementedError):
        T.class_log_probs_fwd(torch.zeros(3, 4), None, 0, -100)


def test_tensors_that_dispatch_to_python_are_refused():
    """Their memory is not the one they show (outputs would be left unwritten); fake tensors are the exception."""
    class Wrapped(torch.Tensor):
        @staticmethod
        def __new__(cls, t):
            return torch.Tensor._make_wrapper_subclass(cls, t.shape, dtype=t.dtype)

        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            raise NotImplementedError
    for call in (lambda: TO.group_norm_act_fwd(Wrapped(torch.zeros(2, 3, 4)), None, None, 2, 1e-5, "none"),
                 lambda: TO.class_log_probs_fwd(Wrapped(torch.zeros(3, 4)), None, 0, -100)):
        with pytest.raises(TypeError, match="plain tensors"):
            call()


def _negated(t):
    """t as a view whose memory holds -t."""
    v = torch.complex(torch.zeros_like(t), -t).conj().imag
    assert v.is_neg() and torch.equal(v, t)
    return v


def test_views_that_hold_their_negative_are_copied_or_refused():
    from erfnet_pytorch_amd import optim
    z = torch.randn(3, 5)
    assert torch.equal(TO.class_layout(_negated(z))[0], z) and not TO.class_layout(_negated(z))[0].is_neg()
    p = torch.nn.Parameter(torch.zeros(6))
    w = optim._host.ParamWatch()
    p.grad = torch.view_as_real(torch.complex(torch.zeros(6), torch.ones(6)))[:, 1].contiguous()
    w.bind([[p]])
    assert [w.look([[p]]) for _ in range(2)] == [1, 0] and w.copied() == []
    p.grad = torch._neg_view(p.grad)                        # the same address
    assert w.look([[p]]) == 1 and w.copied() == [0] and w.look([[p]]) == 1
    with pytest.raises(ValueError, match="negative"):
        optim.AdamW([torch.nn.Parameter(_negated(torch.ones(4)))])


@pytest.mark.gpu
def test_views_that_hold_their_negative_give_what_their_values_give():
    from erfnet_pytorch_amd.loss import class_log_probs
    from erfnet_pytorch_amd.norm import group_norm_act
    from erfnet_pytorch_amd.optim import AdamW
    x, dy, w, b = (torch.randn(*s, device="cuda") for s in ((2, 8, 6, 10), (2, 8, 6, 10), (8,), (8,)))
    t = torch.randint(0, 8, (2, 6, 10), device="cuda")

    def run(view):
        xs, ws, bs = (view(v).detach().requires_grad_() for v in (x, w, b))
        y = group_norm_act(xs, 2, ws, bs, activation="silu")
        out = class_log_probs(xs, t, top_k=2)
        g = torch.autograd.grad([y, out.log_prob, out.top_log_probs], [xs, ws, bs], [view(dy), view(dy[:, 0].clone()), view(dy[:, :2].clone())])
        p = torch.nn.Parameter(b.clone())
        p.grad = view(w)
        AdamW([p]).step()
        return [y, *out, *g, p, *TO.group_norm_act_fwd(view(x.movedim(1, -1).contiguous()), view(w), view(b), 2, 1e-5, "none")]
    want = run(lambda v: v)
    for view in (lambda v: torch._neg_view(-v), lambda v: torch._neg_view(-v.repeat_interleave(2, -1))[..., ::2]):
        assert all(torch.equal(u, v) for u, v in zip(want, run(view)))


def test_forward_mode_differentiation_is_refused():
    """No tangent on the outputs would count as a derivative of 0."""
    import torch.autograd.forward_ad as fa
    from torch._subclasses.fake_tensor import FakeTensorMode
    from erfnet_pytorch_amd.loss import class_log_probs
    from erfnet_pytorch_amd.norm import group_norm_act
    with FakeTensorMode(), fa.dual_level():
        x, w = torch.empty(2, 8, 4, 4, device="cuda"), torch.empty(8, device="cuda")
        for leaf in (False, True):
            dx, dw = (fa.make_dual(t.clone().requires_grad_(leaf), torch.empty_like(t)) for t in (x, w))
            for call in (lambda: group_norm_act(dx, 2), lambda: group_norm_act(x, 2, dw, w), lambda: group_norm_act(x, 2, w, dw),
                         lambda: class_log_probs(dx, top_k=1)):
                for mode in (torch.enable_grad, torch.no_grad):
                    with mode(), pytest.raises(NotImplementedError, match="forward-mode"):
                        call()
        assert group_norm_act(x, 2, w).shape == x.shape and class_log_probs(x).entropy.shape == (2, 4, 4)


@pytest.mark.gpu
def test_outputs_may_be_written_in_place():
    """As torch's own: h = norm(x); h += residual."""
    from erfnet_pytorch_amd.loss import class_log_probs
    from erfnet_pytorch_amd.norm import group_norm_act
    x, r, dy = (torch.randn(2, 8, 6, 10, device="cuda").contiguous(memory_format=torch.channels_last) for _ in range(3))
    grads = []
    for inplace in (False, True):
        xs = x.clone().requires_grad_()
        y = group_norm_act(xs, 2)
        y = y.add_(r).mul_(2.0) if inplace else (y + r) * 2.0
        out = class_log_probs(xs, torch.zeros(2, 6, 10, dtype=torch.int64, device="cuda"), top_k=2)
        lp, top = (out.log_prob.mul_(3.0), out.top_log_probs.mul_(2.0)) if inplace else (out.log_prob * 3.0, out.top_log_probs * 2.0)
        grads.append(torch.autograd.grad((y * dy).sum() + lp.sum() + top.sum(), xs)[0])
    assert torch.equal(*grads)


@pytest.mark.gpu
def test_opcheck_against_the_device_kernels():
    checks = ("test_schema", "test_faketensor")
    x, dy, w, b = (torch.randn(*s, device="cuda") for s in ((2, 8, 16, 24), (2, 8, 16, 24), (24,), (24,)))
    torch.library.opcheck(T.group_norm_act_fwd.default, (x, w, b, 4, 1e-5, "silu"), test_utils=checks)
    y, stats = T.group_norm_act_fwd(x, w, b, 4, 1e-5, "silu")
    torch.library.opcheck(T.group_norm_act_bwd.default, (dy, x, w, b, stats, 4, "silu"), test_utils=checks)
    for z in (torch.randn(2, 20, 8, 16, device="cuda"), torch.randn(5, 1000, device="cuda"),
              torch.randn(2, 20, 8, 16, device="cuda").contiguous(memory_format=torch.channels_last)):
        t = torch.randint(0, 20, (z.shape[0], *z.shape[2:]), device="cuda")
        torch.library.opcheck(T.class_log_probs_fwd.default, (z, t, 3, -100), test_utils=checks)
        lp, ent, st, top, idx = T.class_log_probs_fwd(z, t, 3, -100)
        torch.library.opcheck(T.class_log_probs_bwd.default, (z, t, st, ent, idx, lp, ent, top, -100), test_utils=checks)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(3, 40, 5, 7), (50, 12), (50, 100), (9, 1200), (66000, 20), (2, 40, 4, 6)])
@pytest.mark.parametrize("k", [4, 12])
def test_alternatives_outside_the_classes_have_no_class_of_their_own(shape, k):
    """dz_j = gl ([j = t] - p) + sum_k gk ([j = i_k] - p): such a k gives -p gk alone, in every plan, and nothing beside dz is written.
    Zero logits: p = 1 / C.  Their stats are set here (0, and log C rounded once), so a term's only errors are the exponential's
    (|log p| 3 U + 4 U) p, and one rounding per addition: k + 3 of them."""
    n, c = shape[:2]
    last = shape == (2, 40, 4, 6)
    z = torch.zeros(shape, device="cuda")
    z = z.contiguous(memory_format=torch.channels_last) if last else z
    pos = (n, *shape[2:])
    gen = torch.Generator().manual_seed(5)
    t = torch.randint(0, c, pos, generator=gen)
    gl, gk = torch.randn(pos, generator=gen), torch.randn((n, k, *shape[2:]), generator=gen)
    index = torch.randint(0, c, gk.shape, generator=gen)
    for value, place in ((-1, 1), (c, 2), (2 ** 40, 3), (-2 ** 40, 0)):
        index[:, place] = value
    stats = torch.stack([torch.zeros(pos), torch.full(pos, float(c)).log()])
    dz = T.class_log_probs_bwd(z, t.cuda(), stats.cuda(), torch.zeros(pos, device="cuda"), index.cuda(), gl.cuda(), None, gk.cuda(), -100)
    rows = lambda x: x.movedim(1, -1).reshape(-1, x.shape[1])                                                      # noqa: E731
    want, size = torch.zeros(t.numel(), c, dtype=torch.float64), torch.zeros(t.numel(), c, dtype=torch.float64)
    own = torch.cat([gl.reshape(-1, 1), rows(gk)], 1).double()
    at = torch.cat([t.reshape(-1, 1), rows(index)], 1)
    live = (at >= 0) & (at < c)
    want.scatter_add_(1, torch.where(live, at, 0), torch.where(live, own, 0.0))
    size.scatter_add_(1, torch.where(live, at, 0), torch.where(live, own.abs(), 0.0))
    want, size = want - own.sum(1, keepdim=True) / c, size + own.abs().sum(1, keepdim=True) / c
    assert dz.is_contiguous(memory_format=torch.channels_last) if last else dz.is_contiguous()
    assert ((rows(dz).cpu().double() - want).abs() <= (k + 3 + 4 + 3 * math.log(c)) * U * size).all()


def _step_reference(x, params, t, groups):
    """Loss and gradients of the step below in float64 on the CPU, through torch's own group_norm and log_softmax."""
    w1, gamma, beta, w2 = (p.detach().cpu().double().requires_grad_() for p in params)
    h = x.cpu().double().permute(0, 2, 3, 1) @ w1
    h = torch.nn.functional.silu(torch.nn.functional.group_norm(h.permute(0, 3, 1, 2), groups, gamma, beta, 1e-5))
    logp = torch.log_softmax(h.permute(0, 2, 3, 1) @ w2, -1)
    live = (t != -100).double()
    lp = logp.gather(-1, t.clamp_min(0).unsqueeze(-1))[..., 0] * live
    ent = -(logp.exp() * logp).sum(-1)
    loss = (-(lp.sum()) - 0.01 * (ent * live).sum()) / live.sum()
    return loss, torch.autograd.grad(loss, (w1, gamma, beta, w2))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_training_step_of_all_three(bits):
    """features = x W1, group norm + silu, logits = h W2, mean log loss with an entropy bonus, AdamW; channels-last throughout.
    Every gradient is a sum of at most 2 x 24 x 40 positions' terms, each a product of a chain of sums of at most 32 terms and of the
    norm's sums over 24 x 40 x 8 values: 2048 + 8 x 256 additions one after another at the most (far fewer: they are split), so the
    2-norm of the error is at most 4096 U of the gradient's majorant, which |terms| of one sign bound; twice that is allowed."""
    from erfnet_pytorch_amd.loss import class_log_probs
    from erfnet_pytorch_amd.norm import GroupNormAct2d
    from erfnet_pytorch_amd.optim import AdamW
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(2, 16, 24, 40, generator=gen).cuda().contiguous(memory_format=torch.channels_last)
    t = torch.randint(0, 20, (2, 24, 40), generator=gen)
    t[:, :3] = -100
    norm = GroupNormAct2d(4, 32, activation="silu").cuda()
    w1, w2 = (torch.nn.Parameter((torch.randn(*s, generator=gen) / 4).cuda()) for s in ((16, 32), (32, 20)))
    params = [w1, norm.weight, norm.bias, w2]
    opt = AdamW(params, lr=1e-2, weight_decay=1e-2, state_bits=bits)
    for step in (1, 2, 3):
        want_loss, want = _step_reference(x, params, t, 4)
        opt.zero_grad()
        h = norm((x.permute(0, 2, 3, 1) @ w1).permute(0, 3, 1, 2))
        out = class_log_probs((h.permute(0, 2, 3, 1) @ w2).permute(0, 3, 1, 2), t.cuda(), top_k=2)
        live = (t != -100).cuda()
        loss = (-out.log_prob.sum() - 0.01 * (out.entropy * live).sum()) / live.sum()
        loss.backward()
        assert abs(float(loss.detach()) - float(want_loss.detach())) <= 8192 * U * 10
        for p, g in zip(params, want):
            assert float((p.grad.cpu().double() - g).norm()) <= 8192 * U * float(g.norm())
        before = [p.detach().clone() for p in params]
        state = [{k: v.clone() for k, v in opt.state[p].items()} for p in params] if step > 1 else None
        opt.step()
        for i, p in enumerate(params):                     # the update itself, from the gradient that the step had
            g, q = p.grad.double(), before[i].double()
            if state is None:
                m = v = torch.zeros_like(g)
            elif bits == 32:
                m, v = state[i]["exp_avg"].double(), state[i]["exp_avg_sq"].double()
            else:
                each = lambda k: state[i][k].double().repeat_interleave(256)[:p.numel()].view(p.shape)               # noqa: E731
                m = state[i]["exp_avg"].float().double() * each("exp_avg_scale")
                v = (state[i]["exp_avg_sq_root"].float().double() * each("exp_avg_sq_root_scale")) ** 2
            m, v = 0.9 * m + 0.1 * g, 0.999 * v + 0.001 * g * g
            u = 1e-2 / (1 - 0.9 ** step) * m / ((v / (1 - 0.999 ** step)).sqrt() + 1e-8)
            # 16 roundings of u and of its cancelling moment (|0.9 m| + |0.1 g| <= 20 |u|'s scale), 3 of p: see the optimizer's own tests
            assert ((p.double() - (q * (1 - 1e-4) - u)).abs() <= 64 * U * (q.abs() + 1e-2 * 10)).all()
        assert out.top_log_probs.shape == (2, 2, 24, 40)


@pytest.mark.gpu
def test_the_network_trains_on_label_log_probabilities_with_adamw():
    """ERFNet's logits through class_log_probs: the gradient is the cross entropy's, and AdamW's update reaches the packed weights of
    the next forward pass."""
    from erfnet_pytorch_amd import erfnet as E, synthetic as S
    from erfnet_pytorch_amd.loss import CrossEntropyLoss2d, class_log_probs
    from erfnet_pytorch_amd.optim import AdamW
    model = E.ERFNet(20)
    S.load_synthetic(model)
    model = model.cuda().eval()                             # running statistics, no dropout: the same logits every time
    x = S.synthetic_images(2, 64, 128, seed=1).cuda()
    t = S.synthetic_labels(2, 64, 128, 20, seed=1).cuda().view(2, 64, 128)
    opt = AdamW(model.parameters(), lr=1e-3, state_bits=8)
    logits = model(x)
    loss = -class_log_probs(logits, t).log_prob.mean()
    d1, = torch.autograd.grad(loss, logits, retain_graph=True)
    d2, = torch.autograd.grad(CrossEntropyLoss2d()(logits, t), logits, retain_graph=True)
    # each entry (p - [j = t]) / count: log p to 100 U at logits below 100 either way, the exponentials of the cross entropy another 100 U
    assert (d1 - d2).abs().max() <= 400 * U * 2 / t.numel()
    loss.backward()
    with torch.no_grad():
        before = model(x)
    opt.step()
    assert all(p.isfinite().all() for p in model.parameters())
    with torch.no_grad():
        after = model(x)
    fresh = E.ERFNet(20)
    fresh.load_state_dict(model.state_dict())
    with torch.no_grad():
        again = fresh.cuda().eval()(x)
    assert not torch.equal(before, after) and torch.equal(after, again)
