"""loss.class_log_probs (log probability, entropy, top alternatives of labels) against the definition in 64 bits.

Tolerances, U = 2^-24 (half an fp32 step), from the kernel's formula  m = max z, s = sum e^{z - m}, log p = (z - m) - log s,
H = log s - sum e^{z-m} (z - m) / s:
  a term e^y is off by 2 |y| U from y's two roundings and by at most 4 U from the exponential and its use; a partial sum of n terms adds
  U per addition and 4 U per change of its maximum, 5 n in all.  With A = sum p |z - m| and B = sum p (z - m)^2:
  log s: U (5 n + 4 + 2 A + 2 |log s|) =: E;  log p: E + U (|z - m| + 2 |log p|)
  H: (log s's) + U (5 n + 8) A + 2 U B + E A + 2 U H
  dz: with w = G + gh (log p + H): |p w| (off(log p) + 8 U) + p |gh| (off(log p) + off(H) + 4 U (|log p| + H)) + 4 U (|own| + p (|G| + ...)),
  and half a step of the type; the hardware's exponential gives 0 for results below 2^-126, the smallest normal number, which takes
  up to 2^-126 |w| from p w.  n: additions one after another, the class count for planes, C / 64 + 32 for rows.
"""
import math

import pytest
import torch

U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8}


def _ref(z, target, k, ignore=-100):
    """(log_prob, entropy, top, index) of float64 logits [R, C], differentiable, by torch's own log_softmax on the CPU."""
    logp = torch.log_softmax(z, 1)
    t = target.clamp(0, z.shape[1] - 1)
    lp = torch.where(target == ignore, torch.zeros((), dtype=z.dtype), logp.gather(1, t[:, None])[:, 0])
    p = logp.exp()
    ent = -(p * torch.where(p > 0, logp, torch.zeros((), dtype=z.dtype))).sum(1)
    index = z.detach().sort(dim=1, descending=True, stable=True)[1][:, :k]
    return lp, ent, logp.gather(1, index), index


def _tolerances(z, n):
    """off(log p) [R, C], off(H) [R] of float64 logits whose rows have a finite logit."""
    m = z.max(1, keepdim=True)[0]
    y = (z - m).clamp_min(-1e30)
    p = torch.softmax(z, 1)
    logp = torch.log_softmax(z, 1).clamp_min(-1e30)
    logs = (z - m).exp().sum(1).log()
    a, b = (p * y.abs()).sum(1), (p * y * y).sum(1)
    h = -(p * logp).sum(1)                                  # p = 0 where logp was cut off
    e = U * (5 * n + 4 + 2 * a + 2 * logs.abs())
    return e[:, None] + U * (y.abs() + 2 * logp.abs()), e + U * (5 * n + 8) * a + 2 * U * b + e * a + 2 * U * h


def _close(got, want, tol):
    return (got == want) | ((got - want).abs() <= tol)


def _to_rows(t, k_axis=False):
    """[N, C, ...] -> [R, C] (class axis last), [N, ...] -> [R]."""
    if k_axis:
        return t.movedim(1, -1).reshape(-1, t.shape[1])
    return t.reshape(-1)


def _logits(shape, dtype, layout, seed, spread=3.0, shift=0.0):
    gen = torch.Generator().manual_seed(seed)
    z = (spread * torch.randn(shape, generator=gen) + shift).to(dtype)
    if layout == "channels_last":
        return z.cuda().contiguous(memory_format=torch.channels_last)
    if layout == "padded":                                    # rows further apart than C, first one off the 16-byte grid
        big = torch.full((shape[0], shape[1] + 5), 99.0, dtype=dtype).cuda()
        big[:, 1:1 + shape[1]] = z.cuda()
        return big[:, 1:1 + shape[1]]
    if layout == "sliced":                                    # a run of classes and images of a larger map
        big = torch.full((shape[0] + 1, shape[1] + 2, *shape[2:]), 99.0, dtype=dtype).cuda()
        big[1:, 1:-1] = z.cuda()
        return big[1:, 1:-1]
    if layout == "transposed":                                # no layout of its own: copied
        return z.movedim(1, 0).contiguous().cuda().movedim(0, 1)
    return z.cuda()


def _check(z, target, k, grads=True, seed=0):
    from erfnet_pytorch_amd.loss import class_log_probs
    c = z.shape[1]
    rows_layout = z.dim() == 2 or z.is_contiguous(memory_format=torch.channels_last) if z.dim() in (2, 4) else False
    n = c / 64 + 32 if rows_layout else c
    z = z.detach().requires_grad_(grads)
    out = class_log_probs(z, target, top_k=k)
    zr = _to_rows(z.detach().cpu().double(), True).requires_grad_()
    tr = _to_rows(target.cpu())
    lp, ent, top, index = _ref(zr, tr, k)
    off_lp, off_h = _tolerances(zr.detach(), n)
    shape = (z.shape[0], *z.shape[2:])
    assert out.log_prob.shape == shape and out.entropy.shape == shape and out.log_prob.dtype == out.entropy.dtype == torch.float32
    got = _to_rows(out.log_prob.detach().cpu().double())
    live = tr != -100
    assert _close(got, lp.detach(), off_lp.gather(1, tr.clamp_min(0)[:, None])[:, 0])[live].all() and (got[~live] == 0).all()
    assert ((_to_rows(out.entropy.detach().cpu().double()) - ent.detach()).abs() <= off_h).all()
    if k:
        assert out.top_indices.shape == (shape[0], k, *shape[1:]) and out.top_indices.dtype == torch.int64
        assert torch.equal(_to_rows(out.top_indices.cpu(), True), index)
        assert _close(_to_rows(out.top_log_probs.detach().cpu().double(), True), top.detach(), off_lp.gather(1, index)).all()
    else:
        assert out.top_log_probs is None and out.top_indices is None
    if not grads:
        return
    gen = torch.Generator().manual_seed(seed)
    r = zr.shape[0]
    gl, gh, gk = torch.randn(r, generator=gen), torch.randn(r, generator=gen), torch.randn(r, k, generator=gen)
    back = lambda t: t.reshape(shape).cuda()                                                     # noqa: E731
    outs, gs = [out.log_prob, out.entropy], [back(gl), back(gh)]
    if k:
        outs.append(out.top_log_probs)
        gs.append(gk.reshape(*shape, k).movedim(-1, 1).cuda())
    dz, = torch.autograd.grad(outs, z, gs)
    assert dz.shape == z.shape and dz.dtype == z.dtype
    heads = (lp * gl.double()).sum() + (ent * gh.double()).sum() + (top * gk.double()).sum()
    want, = torch.autograd.grad(heads, zr)
    with torch.no_grad():
        logp = torch.log_softmax(zr, 1)
        p = logp.exp()
        size_lp = logp.abs().clamp_max(1e30)
        pull = (gl.double() * live)[:, None].abs() + gk.double().abs().sum(1, keepdim=True)
        w = pull + gh.double()[:, None].abs() * (size_lp + ent[:, None])
        own = torch.zeros_like(p).scatter_add_(1, tr.clamp_min(0)[:, None], (gl.double().abs() * live)[:, None])
        if k:
            own.scatter_add_(1, index, gk.double().abs())
        tol = p * w * (off_lp + 8 * U) + p * gh.double()[:, None].abs() * (off_lp + off_h[:, None] + 4 * U * (size_lp + ent[:, None])) \
            + 4 * U * (own + p * w) + 8 * k * U * (own + p * pull)
        tol = torch.where(p > 0, tol, 4 * U * own) + HALF[z.dtype] * want.abs() + 2.0 ** -125 + 2.0 ** -126 * w
        assert ((_to_rows(dz.cpu().double(), True) - want).abs() <= tol).all()


def _targets(z, seed, ignored=0.2):
    gen = torch.Generator().manual_seed(seed)
    shape = (z.shape[0], *z.shape[2:])
    t = torch.randint(0, z.shape[1], shape, generator=gen)
    t[torch.rand(shape, generator=gen) < ignored] = -100
    return t.cuda()


ROWS = [(1, 1), (3, 2), (700, 20), (5, 33), (2, 64), (4, 1000), (1, 2049), (3, 4097), (300, 4096), (2, 70001), (1, 200000)]
MAPS = [(1, 1, 3, 3), (2, 20, 5, 7), (2, 6, 1, 1), (1, 150, 16, 17), (3, 2, 1, 1000), (2, 20, 32, 64), (1, 33, 128, 130), (2, 6, 512, 516)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["plain", "padded"])
@pytest.mark.parametrize("shape", ROWS)
def test_rows(shape, layout, dtype):
    z = _logits(shape, dtype, layout, 1)
    t = _targets(z, 2)
    for k in sorted({0, min(3, shape[1]), min(32, shape[1])}):
        _check(z, t, k, seed=k)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("classes", [25, 44, 45, 56, 57, 125, 126, 249, 250, 253, 254, 505, 509, 510, 1017, 1018, 1021, 1022, 2041, 2045, 4089, 4090])
def test_rows_at_the_ends_of_every_plan(classes, dtype):
    """The largest and smallest rows of the threads and of each team, between NaN: what lies beside a row has no effect on it."""
    z = _logits((9, classes), dtype, "plain", classes)
    room = torch.full((9, classes + 3), float("nan"), dtype=dtype, device="cuda")
    room[:, 1:classes + 1] = z
    for k in (0, 3):
        _check(room[:, 1:classes + 1], _targets(z, classes), k)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(65536, 1), (65537, 2), (65700, 9), (65791, 20), (65536, 40), (65536, 41), (65600, 80), (1, 20, 256, 257)])
def test_many_rows_of_few_classes(shape, dtype):
    """The workgroup that works 256 rows off in LDS, its last one in part, and rows just too long or too many alternatives for it;
    channels-last maps are such rows.  Ignored positions full of NaN get 0 and leave their neighbours alone."""
    from erfnet_pytorch_amd.loss import class_log_probs
    z = _logits(shape, dtype, "channels_last" if len(shape) > 2 else "plain", 31)
    t = _targets(z, 32)
    for k in sorted({0, min(2, shape[1]), min(5, shape[1]), min(9, shape[1])}):
        _check(z, t, k, seed=k)
    rows = z.movedim(1, -1).reshape(-1, shape[1])
    want = torch.autograd.grad(class_log_probs(z.requires_grad_(), t).log_prob.sum(), z)[0]
    holes = torch.where((t == -100).reshape(-1, 1), torch.full_like(rows, float("nan")), rows).view(shape[0], *shape[2:], shape[1]).movedim(-1, 1)
    got = torch.autograd.grad(class_log_probs(holes.requires_grad_(), t).log_prob.sum(), holes)[0]
    assert torch.equal(got, want) and bool((t == -100).any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["plain", "channels_last", "sliced", "transposed"])
@pytest.mark.parametrize("shape", MAPS)
def test_maps(shape, layout, dtype):
    z = _logits(shape, dtype, layout, 3)
    t = _targets(z, 4)
    for k in sorted({0, 1, *(min(j, shape[1]) for j in (2, 3, 5, 32))}):
        _check(z, t, k, seed=k)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2, 20, 9), (2, 20, 2, 3, 4), (0, 7), (2, 7, 0, 3)])
def test_other_numbers_of_axes_and_empty_batches(shape):
    from erfnet_pytorch_amd.loss import class_log_probs
    z = _logits(shape, torch.float32, "plain", 5)
    if z.numel():
        return _check(z, _targets(z, 6), 2)
    z.requires_grad_()
    out = class_log_probs(z, torch.zeros((shape[0], *shape[2:]), dtype=torch.int64, device="cuda"), top_k=3)
    assert out.log_prob.shape == (shape[0], *shape[2:]) and out.top_indices.shape == (shape[0], 3, *shape[2:])
    dz, = torch.autograd.grad(out.entropy.sum() + out.log_prob.sum(), z)
    assert dz.shape == z.shape


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(4, 50), (3, 5000), (2, 20, 6, 8)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_far_from_zero_and_widely_spread_logits(shape, dtype):
    for spread, shift in ((3.0, 1e4), (3.0, -1e4), (200.0, 0.0), (1e-3, 0.0), (1e30, 0.0)):
        z = _logits(shape, dtype, "plain", 7, spread, shift)
        _check(z, _targets(z, 8), 3)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(4, 50), (2, 5000), (2, 20, 6, 8), (1, 20, 8, 130)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_equal_values_go_by_index(shape, dtype):
    """All logits equal; a handful of values only; zeros of both signs."""
    for seed, make in enumerate((lambda z: torch.zeros_like(z), lambda z: (z > 0).to(z.dtype), lambda z: (z * 0.5).round(),
                                 lambda z: torch.where(z > 0, 0.0, -0.0).to(z.dtype))):
        z = make(_logits(shape, dtype, "plain", seed))
        _check(z, _targets(z, 9), 20)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(6, 50), (6, 5000), (1, 20, 2, 3)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masked_classes(shape, dtype):
    """-inf and the type's lowest value in masked places: every second class, all but one, all (-inf: no distribution)."""
    from erfnet_pytorch_amd.loss import class_log_probs
    low = torch.finfo(dtype).min
    z = _logits(shape, dtype, "plain", 11)
    rows = z.movedim(1, -1).reshape(-1, shape[1]).clone()
    rows[0, ::2] = float("-inf")
    rows[1, 1:] = float("-inf")
    rows[2, ::2] = low
    rows[3, 1:] = low
    rows[4, :] = low
    rows[5, :7] = float("-inf")
    rows[5, 7:14] = low
    z = rows.reshape(shape[0], *shape[2:], shape[1]).movedim(-1, 1).contiguous()
    t = torch.ones((shape[0], *shape[2:]), dtype=torch.int64, device="cuda")
    t.view(-1)[1] = 0
    _check(z, t, 5)
    t.view(-1)[1] = 1                                       # a masked target: -inf, and a finite gradient
    z.requires_grad_()
    out = class_log_probs(z, t)
    assert float(out.log_prob.detach().reshape(-1)[1]) == float("-inf") and float(out.entropy.detach().reshape(-1)[1]) == 0.0
    dz, = torch.autograd.grad(out.log_prob.view(-1)[1], z)
    dz = dz.movedim(1, -1).reshape(-1, shape[1])
    assert dz[1, 0] == -1 and dz[1, 1] == 1 and (dz[1, 2:] == 0).all() and (dz[0] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(5, 50), (5, 5000), (1, 20, 1, 5)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_positions_without_a_distribution_and_ignored_ones(shape, dtype):
    """All -inf, +inf, NaN: NaN as log_softmax's, in that position alone; ignored or without a gradient, they give exactly 0."""
    from erfnet_pytorch_amd.loss import class_log_probs
    z = _logits(shape, dtype, "plain", 12)
    rows = z.movedim(1, -1).reshape(-1, shape[1]).clone()
    rows[0, :] = float("-inf")
    rows[1, 5] = float("inf")
    rows[2, 7] = float("nan")
    z = rows.reshape(shape[0], *shape[2:], shape[1]).movedim(-1, 1).contiguous().requires_grad_()
    t = torch.tensor([1, 1, 1, 1, -100], device="cuda").reshape(shape[0], *shape[2:])
    out = class_log_probs(z, t, top_k=4)
    lp, ent, top, index = (a.detach() for a in out)
    lp, ent, top, index = lp.reshape(-1), ent.reshape(-1), top.movedim(1, -1).reshape(-1, 4), index.movedim(1, -1).reshape(-1, 4)
    assert lp[:3].isnan().all() and ent[:3].isnan().all() and top[:3].isnan().all() and lp[3:].isfinite().all() and lp[4] == 0 and ent[3:].isfinite().all()
    assert index[0].tolist() == [0, 1, 2, 3] and index[1, 0] == 5 and index[2, 0] == 7
    t = torch.tensor([-100, -100, -100, 1, -100], device="cuda").reshape(shape[0], *shape[2:])
    g = torch.tensor([0, 0, 0, 1.0, 1.0], device="cuda").reshape(t.shape)
    out = class_log_probs(z, t, top_k=4)
    dz, = torch.autograd.grad([out.log_prob, out.entropy, out.top_log_probs], z,
                              [torch.ones_like(g), g, g.unsqueeze(1).expand(g.shape[0], 4, *g.shape[1:])])
    dz = dz.movedim(1, -1).reshape(-1, shape[1])
    assert (dz[:3] == 0).all() and dz[3:].isfinite().all() and (dz[3] != 0).any() and (dz[4] != 0).any()


@pytest.mark.gpu
def test_targets_outside_the_classes_give_nan_and_another_ignore_index():
    from erfnet_pytorch_amd.loss import class_log_probs
    z = _logits((4, 9), torch.float32, "plain", 13).requires_grad_()
    out = class_log_probs(z, torch.tensor([9, -1, 255, 3], device="cuda"), ignore_index=255)
    assert out.log_prob.detach().isnan().tolist() == [True, True, False, False] and out.log_prob[2] == 0
    dz, = torch.autograd.grad(out.log_prob.sum(), z)
    assert dz[:2].isnan().all() and (dz[2] == 0).all() and dz[3].isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(5, 9), (5, 50), (5, 5000), (65600, 20), (1, 20, 1, 5), (2, 9, 640, 512)])
@pytest.mark.parametrize("last", [False, True])
def test_targets_outside_the_classes_without_a_gradient_give_none(shape, last):
    """Such positions masked by the caller: exactly 0 in every plan, or what the other outputs' gradients give alone."""
    from erfnet_pytorch_amd.loss import class_log_probs
    z = _logits(shape, torch.float32, "channels_last" if last and len(shape) == 4 else "plain", 15).requires_grad_()
    pos = (shape[0], *shape[2:])
    t = torch.zeros(pos, dtype=torch.int64, device="cuda")
    flat = t.view(-1)
    flat[0], flat[1], flat[2], flat[-1] = -1, shape[1], 2 ** 40, -7
    g = torch.ones(pos, device="cuda")
    for i in (0, 2, -1):
        g.view(-1)[i] = 0
    h = torch.zeros(pos, device="cuda")
    h.view(-1)[2] = 1.0
    out = class_log_probs(z, t)
    dz, = torch.autograd.grad([out.log_prob, out.entropy], z, [g, h])
    dh, = torch.autograd.grad(class_log_probs(z).entropy, z, h)
    dz, dh = (d.movedim(1, -1).reshape(-1, shape[1]) for d in (dz, dh))
    assert (dz[0] == 0).all() and dz[1].isnan().all() and torch.equal(dz[2], dh[2]) and (dz[-1] == 0).all() and dz[3].isfinite().all()


@pytest.mark.gpu
def test_without_target_and_partial_gradients():
    from erfnet_pytorch_amd.loss import class_log_probs
    z = _logits((3, 30), torch.float32, "plain", 14).requires_grad_()
    out = class_log_probs(z, top_k=2)
    assert out.log_prob is None
    d1, = torch.autograd.grad(out.entropy.sum(), z, retain_graph=True)
    d2, = torch.autograd.grad(out.top_log_probs.sum(), z)
    zr = z.detach().cpu().double().requires_grad_()
    _, ent, top, _ = _ref(zr, torch.zeros(3, dtype=torch.int64), 2)
    w1, = torch.autograd.grad(ent.sum(), zr, retain_graph=True)
    w2, = torch.autograd.grad(top.sum(), zr)
    # 32 + 30 / 64 additions, log p and H below 12: every factor within 2000 U of its value
    assert (d1.cpu() - w1).abs().max() <= 2000 * U * 24 and (d2.cpu() - w2).abs().max() <= 2000 * U * 4
    with torch.no_grad():
        assert not class_log_probs(z).entropy.requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("classes,k,rows", [(60, 0, 2 ** 27 + 500), (600, 2, 2 ** 26 + 500), (1500, 1, 2 ** 24 + 500), (4500, 1, 2 ** 22 + 500)])
def test_more_rows_than_one_launch_takes(classes, k, rows):
    """Rows that overlap in memory (the next one starts a class later), by teams of 8, 16 and 64 and by workgroups: around the seams of the
    launches the bits of a call on those rows alone."""
    from erfnet_pytorch_amd import train_ops as TO
    buf = torch.randn(rows + classes, device="cuda").to(torch.bfloat16)
    z, t = buf.as_strided((rows, classes), (1, 1)), torch.randint(0, classes, (rows,), device="cuda")
    lp, ent, stats, top, idx = TO.class_log_probs_fwd(z, t, k, -100)
    seam = rows - 500
    here = slice(seam - 40, seam + 40)
    part = TO.class_log_probs_fwd(z[here], t[here], k, -100)
    for whole, alone in ((lp[here], part[0]), (ent[here], part[1]), (stats[:, here], part[2]), (top[here], part[3]), (idx[here], part[4])):
        assert torch.equal(whole, alone)
    assert not torch.isnan(lp).any() and float(lp.max()) <= 0
    if classes > 60:                                        # (of a gradient of 16 GB a sample is enough)
        return
    g = torch.randn(rows, device="cuda")
    dz = TO.class_log_probs_bwd(z, t, stats, ent, idx, g, None, None, -100)
    assert torch.equal(dz[here], TO.class_log_probs_bwd(z[here], t[here], part[2], part[1], part[4], g[here], None, None, -100))


@pytest.mark.gpu
@pytest.mark.parametrize("shape,stride", [((4, 1000), (2 ** 31, 1)), ((4, 40), (2 ** 31, 1)), ((2, 20, 64), (20 * 2 ** 27, 2 ** 27, 1))])
def test_offsets_that_pass_32_bits(shape, stride):
    """Rows, and planes, so far apart: the bits of a compact copy."""
    from erfnet_pytorch_amd import train_ops as TO
    room = torch.empty(sum((n - 1) * s for n, s in zip(shape, stride)) + 1, dtype=torch.bfloat16, device="cuda")
    small = _logits(shape, torch.bfloat16, "plain", 3)
    z = room.as_strided(shape, stride).copy_(small)
    t = torch.randint(0, shape[1], (shape[0], *shape[2:]), device="cuda")
    outs = [TO.class_log_probs_fwd(v, t, 3, -100) for v in (z, small)]
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    g, top = torch.randn(t.shape, device="cuda"), torch.randn(outs[0][3].shape, device="cuda")
    dz = [TO.class_log_probs_bwd(v, t, o[2], o[1], o[4], g, g, top, -100) for v, o in zip((z, small), outs)]
    assert torch.equal(*dz)


@pytest.mark.gpu
@pytest.mark.parametrize("shape,k", [((40, 9), 5), ((40, 60), 3), ((40, 60), 20), ((9, 300), 32), ((9, 1200), 32), ((5, 5000), 32), ((2, 20, 4, 6), 2), ((2, 20, 4, 6), 12)])
def test_alternatives_that_name_a_class_more_than_once(shape, k):
    """The backward pass takes the classes as they are given: the same one several times, and the target's, get every gradient.

    p is off by at most (2 |log p| + 8) U of itself, the sums of k gradients by k U: in all (2 max |log p| + k + 16) U of
    (|gl| + sum |gk|) (1 + p) + |gh| p (|log p| + H)."""
    from erfnet_pytorch_amd import train_ops as TO
    z = _logits(shape, torch.float32, "plain", 21, spread=1.0)
    n, c = shape[:2]
    pos = (n, *shape[2:])
    gen = torch.Generator().manual_seed(22)
    t = torch.randint(0, c, pos, generator=gen)
    idx = torch.randint(0, c, (n, k, *shape[2:]), generator=gen)
    idx[:, 1] = idx[:, 0]
    idx[: n // 2, k - 1] = t[: n // 2]
    gl, gh, gk = torch.randn(pos, generator=gen), torch.randn(pos, generator=gen), torch.randn(idx.shape, generator=gen)
    _, ent, stats, _, _ = TO.class_log_probs_fwd(z, t.cuda(), 0, -100)
    got = _to_rows(TO.class_log_probs_bwd(z, t.cuda(), stats, ent, idx.cuda(), gl.cuda(), gh.cuda(), gk.cuda(), -100).cpu().double(), True)
    lp = torch.log_softmax(_to_rows(z.cpu().double(), True), -1)
    p, h = lp.exp(), -(lp.exp() * lp).sum(-1, keepdim=True)
    tr, ir, lr, hr, kr = t.reshape(-1, 1), _to_rows(idx, True), gl.double().reshape(-1, 1), gh.double().reshape(-1, 1), _to_rows(gk.double(), True)
    want = torch.zeros_like(p).scatter_add_(1, tr, lr).scatter_add_(1, ir, kr) - p * (lr + kr.sum(-1, keepdim=True)) - hr * p * (lp + h)
    size = (lr.abs() + kr.abs().sum(-1, keepdim=True)) * (1 + p) + hr.abs() * p * (lp.abs() + h)
    assert ((got - want).abs() <= (2 * float(lp.abs().max()) + k + 16) * U * size).all()


@pytest.mark.gpu
def test_second_derivatives_are_refused():
    from erfnet_pytorch_amd.loss import class_log_probs
    z = _logits((3, 30), torch.float32, "plain", 17).requires_grad_()
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(class_log_probs(z).entropy.sum(), z, create_graph=True)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(3, 11), (1, 11, 1, 3)])
def test_gradient_against_differences(shape):
    """(f(z + h) - f(z - h)) / 2h with h = 2^-6: truncated at h^2 / 6 |f'''|, |f'''| <= 40 for log p and H of logits this flat
    (third derivatives are sums of at most 6 products of numbers up to log 11 + 2), rounded by 2 * 2000 U / 2h."""
    from erfnet_pytorch_amd.loss import class_log_probs
    z = _logits(shape, torch.float32, "plain", 15, 0.5)
    t = _targets(z, 16, 0.0)
    zz = z.clone().requires_grad_()
    out = class_log_probs(zz, t)
    grads = [torch.autograd.grad(f.sum(), zz, retain_graph=True)[0] for f in (out.log_prob, out.entropy)]
    h = 2.0 ** -6
    for c in range(shape[1]):
        ends = []
        for s in (h, -h):
            moved = z.clone()
            moved[:, c] += s
            o = class_log_probs(moved, t)
            ends.append((o.log_prob, o.entropy))
        for f, g in enumerate(grads):
            diff = (ends[0][f].double() - ends[1][f].double()) / (2 * h)
            assert (diff - g[:, c].double()).abs().max() <= h * h / 6 * 40 + 4000 * U / (2 * h)


@pytest.mark.gpu
def test_rows_of_the_gradient_do_not_touch_what_lies_between_them():
    from erfnet_pytorch_amd import _lib, ops, train_ops
    n, c, s = 5, 37, 48
    gen = torch.Generator().manual_seed(19)
    z, t = torch.randn(n, s, generator=gen).cuda(), torch.randint(0, c, (n,), generator=gen).cuda()
    d, one = torch.full((n, s), 7.0, device="cuda"), torch.ones(n, device="cuda")
    _, ent, stats, _, index = train_ops.class_log_probs_fwd(z[:, :c], t, 0, -100)
    want = train_ops.class_log_probs_bwd(z[:, :c], t, stats, ent, index, one, None, None, -100)
    _lib.call("erf_class_log_probs_bwd", z.data_ptr(), _lib.F32, n, c, 1, s, 1, t.data_ptr(), -100, stats.data_ptr(), ent.data_ptr(), one.data_ptr(),
              0, 0, 0, 0, d.data_ptr(), s, 1, ops._stream())
    assert torch.equal(d[:, :c], want) and (d[:, c:] == 7.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 70001), (40, 1000), (2, 20, 16, 32)])
def test_captured_calls_and_another_stream(shape):
    """Forward and backward captured together, replayed on new inputs with eager calls between; two graphs at once; a side stream."""
    from erfnet_pytorch_amd.loss import class_log_probs

    def both(z, t, g):
        out = class_log_probs(z, t, top_k=4)
        dz, = torch.autograd.grad([out.log_prob, out.entropy], z, [g, g])
        return [a.detach() for a in out] + [dz]
    z = [_logits(shape, torch.bfloat16, "plain", 20 + i).requires_grad_() for i in range(2)]
    t = [_targets(z[i], 30 + i) for i in range(2)]
    g = torch.randn(t[0].shape, device="cuda")
    both(z[0], t[0], g)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, capture_error_mode="thread_local"):
            outs.append(both(z[i], t[i], g))
        graphs.append(gr)
    for rep in range(3):
        for i in range(2):
            with torch.no_grad():
                z[i].copy_(_logits(shape, torch.bfloat16, "plain", 40 + 2 * rep + i))
        for gr in graphs:
            gr.replay()
        want = [both(z[i].detach().clone().requires_grad_(), t[i], g) for i in range(2)]
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(a, b) for a, b in zip(outs[i], want[i]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = both(z[0].detach().clone().requires_grad_(), t[0], g)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(there, want[0]))


# ------------------------------------------------------------------------------------------------ refusals (CPU)
def test_wrong_arguments_are_refused():
    from erfnet_pytorch_amd import train_ops
    from erfnet_pytorch_amd.loss import class_log_probs
    z = torch.zeros(3, 5)
    with pytest.raises(RuntimeError, match="MI355X"):
        class_log_probs(z, torch.zeros(3, dtype=torch.int64))
    def f(z, target, top_k=0):
        return train_ops.class_log_probs_fwd(z, target, top_k, -100)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        f(z.half(), None)
    with pytest.raises(TypeError, match="int64"):
        f(z, torch.zeros(3, dtype=torch.int32))
    for bad in (torch.zeros(4, dtype=torch.int64), torch.zeros(3, 5, dtype=torch.int64)):
        with pytest.raises(ValueError, match="targets of shape"):
            f(z, bad)
    with pytest.raises(ValueError, match="on meta"):
        f(z, torch.zeros(3, dtype=torch.int64, device="meta"))
    with pytest.raises(RuntimeError, match="MI355X"):
        f(z, None)
    for k in (-1, 6):
        with pytest.raises(ValueError, match="top_k"):
            f(z, None, k)
    with pytest.raises(ValueError, match="top_k"):
        f(torch.zeros(1, 100), None, 33)
    for bad in (torch.zeros(3), torch.zeros(3, 0)):
        with pytest.raises(ValueError, match="shape"):
            f(bad, None)
    b = train_ops.class_log_probs_bwd
    t, v, two, index = torch.zeros(3, dtype=torch.int64), torch.zeros(3), torch.zeros(2, 3), torch.zeros(3, 2, dtype=torch.int64)
    for args in ((z, t, torch.zeros(2, 4), v, index, v, None, None), (z, t, two, torch.zeros(4), index, v, None, None),
                 (z, None, two, v, index, v, None, None), (z, t, two, v, index, torch.zeros(4), None, None), (z, t, two, v, index, None, torch.zeros(2), None),
                 (z, t, two, v, index, None, None, torch.zeros(3, 1)), (z, t, two, v, index.int(), None, None, torch.zeros(3, 2)),
                 (z, t, two.double(), v, index, v, None, None), (z, t, two, v, index, v.to("meta"), None, None)):
        with pytest.raises(ValueError):
            b(*args, -100)


def test_abi_refuses_bad_arguments_without_a_gpu():
    from erfnet_pytorch_amd import _lib
    good = [16, 0, 4, 5, 1, 5, 1, 16, -100, 16, 16, 16, 2, 16, 16, 0, 0]
    for i, bad in ((0, 0), (1, 2), (2, 0), (3, 0), (4, 0), (5, -1), (6, 0), (7, 0), (9, 0), (10, 0), (12, 6), (12, -1), (13, 0), (14, 0)):
        args = list(good)
        args[i] = bad
        assert _lib.query("erf_class_log_probs_fwd", *args) == -1, i
    assert _lib.query("erf_class_log_probs_workspace_bytes", 1, 1, 200000, 1, 1, 4) > 0
    assert _lib.query("erf_class_log_probs_fwd", 16, 1, 1, 200000, 1, 200000, 1, 16, -100, 16, 16, 16, 2, 16, 16, 0, 0) == -1      # no workspace
    good = [16, 0, 4, 5, 6, 30, 6, 16, -100, 16, 16, 16, 16, 2, 16, 16, 16, 30, 6, 0]
    for i, bad in ((0, 0), (1, 2), (2, 0), (3, 0), (4, 0), (6, 5), (6, 1), (7, 0), (9, 0), (10, 0), (13, 33), (14, 0), (16, 0), (17, -1), (18, 5), (18, 1)):
        args = list(good)
        args[i] = bad
        assert _lib.query("erf_class_log_probs_bwd", *args) == -1, i


def test_abi_refuses_gradients_that_share_memory_without_a_gpu():
    """Rows closer than C, planes or images on top of each other: two threads would write one place.  (Accepted strides reach a launch,
    which there is no device for here: another status.)"""
    from erfnet_pytorch_amd import _lib
    if torch.cuda.is_available():
        pytest.skip("the accepted calls have no memory behind them")

    def status(n, c, length, dn, dc):
        rows = dc == 1
        return _lib.query("erf_class_log_probs_bwd", 16, 0, n, c, length, c * length, 1 if rows else max(length, 2), 16, -100, 16, 16, 16, 0, 0, 0, 0, 16, dn, dc, 0)
    for bad in ((2, 5, 1, 0, 1), (2, 5, 1, 4, 1), (2, 5, 6, 29, 6), (2, 5, 6, 0, 6), (2, 5, 6, 5, 100), (3, 5, 6, 6, 17), (2, 1, 6, 5, 6),
                (2, 2 ** 28, 6, 2 ** 62, 2 ** 62)):
        assert status(*bad) == -1, bad
    for good in ((1, 5, 1, 0, 1), (2, 5, 1, 5, 1), (2, 5, 1, 9, 1), (2, 5, 6, 30, 6), (1, 5, 6, 0, 6), (3, 5, 6, 6, 18), (2, 1, 6, 6, 6), (2, 2 ** 28, 6, 2 ** 61, 2 ** 62)):
        assert status(*good) == -3, good


def test_layouts_are_recognised():
    from erfnet_pytorch_amd.train_ops import class_layout as whole

    def class_layout(t):
        z, n, c, length, sn, sc, rows = whole(t)
        return z, n, c, length, sn, sc
    z = torch.zeros(2, 5, 3, 4)
    assert class_layout(z)[1:6] == (2, 5, 12, 60, 12)
    assert class_layout(z.contiguous(memory_format=torch.channels_last))[1:6] == (24, 5, 1, 5, 1)
    assert class_layout(z[:, 1:3])[1:6] == (2, 2, 12, 60, 12)
    assert class_layout(z.transpose(2, 3))[0].is_contiguous()
    assert class_layout(torch.zeros(4, 9)[:, 2:7])[1:6] == (4, 5, 1, 9, 1)
    assert class_layout(torch.zeros(1, 1, 3, 4))[1:6] == (1, 1, 12, 12, 12)
    assert class_layout(torch.zeros(2, 5, 1, 1))[1:6] == (2, 5, 1, 5, 1)
    assert class_layout(torch.zeros(3, 8, 1, 1)[:, 1:7])[1:6] == (3, 6, 1, 8, 1)
    assert class_layout(torch.zeros(3, 8, 1, 2)[..., :1])[1:6] == (3, 8, 1, 8, 1)
    assert class_layout(torch.zeros(3, 1, 1, 1))[1:6] == (3, 1, 1, 1, 1)
    assert class_layout(torch.zeros(4, 3).t())[1:6] == (3, 4, 1, 4, 1)
    assert math.prod(class_layout(torch.zeros(0, 7, 3, 4))[1:4:2]) == 0
