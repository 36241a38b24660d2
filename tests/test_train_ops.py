"""Layer norm, token log probabilities and AdamW (functional.layer_norm, functional.log_probs, optim.AdamW) against plain
formulas in 64 bits, and their refusals.

Tolerances are bounds of first-order rounding error, with u = 2^-24 the largest relative error of one fp32 rounding.
A sum over a row is at most 16 serial additions in a thread, 6 across a wave and 16 across a block's waves: with the
products before it, under 48 roundings on the longest path, so a sum errs by at most 48 u of the sum of magnitudes; 64 u
leaves room for the few operations behind it.  A result stored in bf16 adds its own rounding, at most 2^-8 of itself."""
import ctypes as C

import pytest
import torch

U = 2.0 ** -24
DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
gpu = pytest.mark.gpu


def half_step(t):
    return 0.0 if t == torch.float32 else torch.finfo(t).eps / 2


def within(got, ref, tol, what):
    got, ref = got.double().cpu(), ref.double().cpu()
    tol = torch.as_tensor(tol, dtype=torch.float64).cpu().expand(ref.shape)
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    both = torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), what
    assert torch.equal(got[torch.isinf(ref)], ref[torch.isinf(ref)]), what
    assert torch.isfinite(got[both]).all(), what
    off = (got - ref).abs()[both] - tol[both]
    assert off.numel() == 0 or off.max() <= 0, (what, float(off.max()), float((got - ref).abs()[both].max()))



# ================================================================================ layer norm
def norm_case(rows, c, kind, level=0.0, seed=0):
    g = torch.Generator().manual_seed(1000 * rows + c + seed)
    x = (torch.randn(rows, c, generator=g) * 1.5 + level).to(kind)
    gy = torch.randn(rows, c, generator=g).to(kind)
    w = 1 + 0.3 * torch.randn(c, generator=g)
    b = 0.3 * torch.randn(c, generator=g)
    return x, gy, w, b


def norm_reference(x, gy, w, b, eps):
    """y, dx, dw, db in float64 and, for each, the sum of magnitudes its rounding error is proportional to."""
    x, gy = x.double(), gy.double()
    w = torch.ones(x.shape[1], dtype=torch.float64) if w is None else w.double()
    b = torch.zeros(x.shape[1], dtype=torch.float64) if b is None else b.double()
    mean = x.mean(1, keepdim=True)
    d = x - mean
    r = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + eps)
    h = d * r
    gw = gy * w
    c1, c2 = gw.mean(1, keepdim=True), (gw * h).mean(1, keepdim=True)
    level = x.abs().mean(1, keepdim=True) * r            # error of the mean, in units of the row's spread
    y = h * w + b
    y_mag = w.abs() * (level + h.abs() * (2 + level)) + b.abs()
    dx = r * (gw - c1 - h * c2)
    m1, m2 = gw.abs().mean(1, keepdim=True), (gw * h).abs().mean(1, keepdim=True)
    hm = h.abs() * (2 + level) + level                   # magnitude behind xhat's own error
    dx_mag = r * (2 + level) * (gw.abs() + m1 + h.abs() * m2) + r * (hm * m2 + h.abs() * (gw.abs() * hm).mean(1, keepdim=True))
    return (y, dx, (gy * h).sum(0), gy.sum(0)), (y_mag, dx_mag, (gy.abs() * (h.abs() + hm)).sum(0), gy.abs().sum(0))


def check_norm(got, x, gy, w, b, eps, what):
    refs, mags = norm_reference(x, gy, w, b, eps)
    for name, o, ref, mag in zip(("y", "dx", "dw", "db"), got, refs, mags):
        if o is None:
            continue
        k = 64 if name in ("y", "dx") else 128          # weight sums: a thread's rows, a wave, a block, 32 + 32 blocks
        stored = half_step(o.dtype)
        within(o.reshape(ref.shape), ref, stored * ref.abs() + k * U * mag * (1 + stored), f"{what} {name}")


NORM_SHAPES = [(1, 1), (3, 1), (1, 5), (33, 1000), (7, 16), (129, 17), (64, 31), (50, 64), (300, 128), (9, 255), (5, 1024),
               (4, 1025), (3, 2047), (6, 4096), (2, 4097), (3, 8191), (2, 16384), (5, 8193), (300, 12001)]


@gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,c", NORM_SHAPES)
def test_layer_norm_rows(rows, c, kind):
    from erfnet_pytorch_amd import functional as hipf
    x, gy, w, b = norm_case(rows, c, TYPES[kind])
    args = [t.to(DEV).requires_grad_() for t in (x, w, b)]
    y = hipf.layer_norm(*args, eps=1e-5)
    assert y.dtype == x.dtype and y.shape == x.shape
    grads = torch.autograd.grad(y, args, gy.to(DEV))
    check_norm((y.detach(), *grads), x, gy, w, b, 1e-5, (rows, c, kind))
    with torch.no_grad():
        assert torch.equal(hipf.layer_norm(*args, eps=1e-5), y)


@gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n,c,h,w_", [(2, 16, 24, 40), (1, 64, 9, 13), (3, 128, 8, 7), (1, 13, 5, 6), (2, 1, 4, 4), (1, 20, 1, 1)])
def test_layer_norm_over_the_channels_of_an_image(n, c, h, w_, kind):
    from erfnet_pytorch_amd import functional as hipf
    x, gy, w, b = norm_case(n * h * w_, c, TYPES[kind], level=2.0)
    image = lambda t: t.view(n, h, w_, c).permute(0, 3, 1, 2)       # noqa: E731
    for xi, gi in ((image(x).to(DEV), image(gy).to(DEV)), (image(x).contiguous().to(DEV), image(gy).contiguous().to(DEV))):
        args = [t.detach().requires_grad_() for t in (xi, w.to(DEV), b.to(DEV))]
        y = hipf.layer_norm(*args, eps=1e-3, dim=1)
        assert y.shape == xi.shape
        dx, dw, db = torch.autograd.grad(y, args, gi)
        rows = lambda t: t.permute(0, 2, 3, 1).reshape(-1, c)       # noqa: E731
        check_norm((rows(y.detach()), rows(dx), dw, db), x, gy, w, b, 1e-3, (n, c, h, w_, kind))


@gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("has_w,has_b", [(False, False), (True, False), (False, True)])
def test_layer_norm_without_weight_or_bias(has_w, has_b, kind):
    from erfnet_pytorch_amd import functional as hipf
    x, gy, w, b = norm_case(70, 96, TYPES[kind])
    w, b = (w if has_w else None), (b if has_b else None)
    args = [None if t is None else t.to(DEV).requires_grad_() for t in (x, w, b)]
    y = hipf.layer_norm(*args)
    grads = iter(torch.autograd.grad(y, [t for t in args if t is not None], gy.to(DEV)))
    got = [None if t is None else next(grads) for t in args]
    check_norm((y.detach(), *got), x, gy, w, b, 1e-5, (has_w, has_b, kind))


@gpu
def test_layer_norm_gradient_of_the_parameters_alone_and_of_x_alone():
    from erfnet_pytorch_amd import functional as hipf
    x, gy, w, b = norm_case(100, 72, torch.float32)
    xd, wd, bd, gd = (t.to(DEV) for t in (x, w, b, gy))
    wd.requires_grad_(), bd.requires_grad_()
    dw, db = torch.autograd.grad(hipf.layer_norm(xd, wd, bd), (wd, bd), gd)
    xd.requires_grad_(), wd.requires_grad_(False), bd.requires_grad_(False)
    dx, = torch.autograd.grad(hipf.layer_norm(xd, wd, bd), xd, gd)
    check_norm((None, dx, dw, db), x, gy, w, b, 1e-5, "separate")


@gpu
def test_layer_norm_level_far_from_zero_keeps_its_variance():
    """Rows at 1000 +- 1.5: E[x^2] - mean^2 in fp32 would have no digit of the variance left."""
    from erfnet_pytorch_amd import functional as hipf
    x, gy, w, b = norm_case(40, 500, torch.float32, level=1000.0)
    args = [t.to(DEV).requires_grad_() for t in (x, w, b)]
    y = hipf.layer_norm(*args)
    check_norm((y.detach(), *torch.autograd.grad(y, args, gy.to(DEV))), x, gy, w, b, 1e-5, "level")


@gpu
def test_layer_norm_constant_rows_and_non_finite_rows():
    from erfnet_pytorch_amd import functional as hipf
    x = torch.randn(6, 40, generator=torch.Generator().manual_seed(3))
    x[1] = 0.75
    x[3, 7] = float("inf")
    x[4, 0] = float("nan")
    y = hipf.layer_norm(x.to(DEV)).cpu()
    assert torch.equal(y[1], torch.zeros(40))
    assert torch.isnan(y[3]).all() and torch.isnan(y[4]).all()
    keep = [0, 2, 5]
    check_norm((y[keep],), x[keep], torch.zeros(3, 40), None, None, 1e-5, "neighbours of a NaN")


@gpu
def test_layer_norm_strided_input_expanded_gradient_and_bf16_parameters():
    from erfnet_pytorch_amd import functional as hipf
    x, gy, w, b = norm_case(24, 64, torch.float32)
    wide = torch.zeros(24, 100, device=DEV)
    wide[:, 20:84] = x.to(DEV)
    xs = wide[:, 20:84].requires_grad_()
    wh, bh = w.bfloat16(), b.bfloat16()
    wd, bd = wh.to(DEV).requires_grad_(), bh.to(DEV).requires_grad_()
    y = hipf.layer_norm(xs, wd, bd)
    dx, dw, db = torch.autograd.grad(y.sum(), (xs, wd, bd))
    assert dw.dtype == torch.bfloat16 and db.dtype == torch.bfloat16
    check_norm((y.detach(), dx, dw, db), x, torch.ones(24, 64), wh.float(), bh.float(), 1e-5, "strided")


@gpu
def test_layer_norm_no_rows():
    from erfnet_pytorch_amd import functional as hipf
    x = torch.zeros(0, 8, device=DEV, requires_grad=True)
    w = torch.ones(8, device=DEV, requires_grad=True)
    y = hipf.layer_norm(x, w)
    dx, dw = torch.autograd.grad(y.sum(), (x, w))
    assert y.shape == (0, 8) and dx.shape == (0, 8) and torch.equal(dw.cpu(), torch.zeros(8))


@gpu
def test_layer_norm_gradient_against_differences():
    """Central differences of the kernel's own forward, step h = 2^-6: fp32 noise of the difference is at most
    64 u (|y| magnitude ~ 4 of 40 terms) / h, the formula's third-order term h^2 times a derivative of order 1."""
    from erfnet_pytorch_amd import functional as hipf
    x, gy, w, b = norm_case(3, 40, torch.float32)
    xd, wd, bd, gd = (t.to(DEV) for t in (x, w, b, gy))
    leaf = xd.clone().requires_grad_()
    dx, = torch.autograd.grad(hipf.layer_norm(leaf, wd, bd), leaf, gd)
    h = 2.0 ** -6
    loss = lambda t: float((hipf.layer_norm(t, wd, bd).double() * gd.double()).sum())     # noqa: E731
    for r, c in ((0, 0), (1, 17), (2, 39)):
        up, down = xd.clone(), xd.clone()
        up[r, c] += h
        down[r, c] -= h
        num = (loss(up) - loss(down)) / (2 * h)
        assert abs(num - float(dx[r, c])) <= 64 * U * 4 * 40 / h + 16 * h * h, (r, c, num, float(dx[r, c]))


@gpu
def test_layer_norm_pointers_of_any_alignment():
    from erfnet_pytorch_amd import functional as hipf
    for kind in TYPES.values():
        x, gy, w, b = norm_case(21, 88, kind)
        buf, bufg = (torch.zeros(21 * 88 + 9, dtype=kind, device=DEV) for _ in range(2))
        for off in (1, 3, 8):
            xs, gs = (t[off:off + 21 * 88].view(21, 88) for t in (buf, bufg))
            xs.copy_(x), gs.copy_(gy)
            args = [t.detach().requires_grad_() for t in (xs, w.to(DEV), b.to(DEV))]
            y = hipf.layer_norm(*args)
            check_norm((y.detach(), *torch.autograd.grad(y, args, gs)), x, gy, w, b, 1e-5, (kind, off))


@gpu
def test_layer_norm_beyond_32_bit_offsets():
    """2^31 + 5120 elements: the last rows equal the same rows by themselves, bit for bit."""
    from erfnet_pytorch_amd import functional as hipf
    rows, c = (1 << 21) + 5, 1024
    x = torch.zeros(rows, c, dtype=torch.bfloat16, device=DEV)
    gy = torch.zeros_like(x)
    tail, gtail, w, b = norm_case(6, c, torch.bfloat16)
    x[-6:], gy[-6:] = tail.to(DEV), gtail.to(DEV)
    w, b = w.to(DEV), b.to(DEV)
    x.requires_grad_()
    y = hipf.layer_norm(x, w, b)
    dx, = torch.autograd.grad(y, x, gy)
    part = tail.to(DEV).requires_grad_()
    yp = hipf.layer_norm(part, w, b)
    dxp, = torch.autograd.grad(yp, part, gtail.to(DEV))
    assert torch.equal(y[-6:], yp) and torch.equal(dx[-6:], dxp)


def test_layer_norm_module_on_the_cpu():
    from erfnet_pytorch_amd.norm import LayerNorm
    x, gy, w, b = norm_case(30, 12, torch.float32)
    m = LayerNorm(12, dim=1)
    with torch.no_grad():
        m.weight.copy_(w), m.bias.copy_(b)
    y = m(x.view(2, 5, 3, 12).permute(0, 3, 1, 2)).permute(0, 2, 3, 1).reshape(30, 12)
    within(y.detach(), norm_reference(x, gy, w, b, 1e-5)[0][0], 1e-5, "module")
    assert list(LayerNorm(4).state_dict()) == ["weight", "bias"] and not LayerNorm(4, affine=False).state_dict()
    with pytest.raises(ValueError):
        LayerNorm(4, dim=0)
    with pytest.raises(ValueError, match="4 channels"):
        LayerNorm(4, affine=False)(torch.zeros(3, 5))
    with pytest.raises(ValueError, match="4 channels"):
        LayerNorm(4, dim=1)(torch.zeros(4))
    # one rounding of the result to bf16 on top of fp32's
    y = m.bfloat16()(x.view(2, 5, 3, 12).permute(0, 3, 1, 2).bfloat16())
    x16, w16, b16 = x.bfloat16(), w.bfloat16(), b.bfloat16()
    want = norm_reference(x16, gy, w16, b16, 1e-5)[0][0]
    got = y.detach().permute(0, 2, 3, 1).reshape(30, 12)
    assert y.dtype == torch.bfloat16 and ((got.double() - want).abs() <= want.abs() * 2.0 ** -8 + 1e-5).all()


@gpu
def test_layer_norm_module_between_blocks():
    """In front of and behind a non_bottleneck_1d: NHWC in and out, gradients through both."""
    from erfnet_pytorch_amd import erfnet_blocks
    from erfnet_pytorch_amd.norm import LayerNorm
    torch.manual_seed(3)
    net = torch.nn.Sequential(LayerNorm(64, dim=1), erfnet_blocks.non_bottleneck_1d(64, 0.0, 1), LayerNorm(64, dim=1))
    x = torch.randn(1, 64, 16, 24)
    want = net(x)
    g = torch.randn_like(want)
    want_grads = torch.autograd.grad(want, list(p for p in net.parameters()), g, allow_unused=True)
    net = net.to(DEV)
    got = net(x.to(DEV))
    got_grads = torch.autograd.grad(got, list(p for p in net.parameters()), g.to(DEV), allow_unused=True)
    # convolutions of 64 x 3 products on both sides: 2e-4 of the largest value, as the blocks' own tests allow
    assert (got.cpu() - want).abs().max() <= 2e-4 * want.abs().max()
    for a, b_ in zip(got_grads, want_grads):
        assert (a is None) == (b_ is None)
        if a is not None:
            assert (a.cpu() - b_).abs().max() <= 1e-3 * b_.abs().max().clamp(min=1e-6)


# ================================================================================ log probabilities
def lp_reference(x, target, k, ignore, g_lp=None, g_h=None, g_top=None):
    """Rows [n, V] in float64: results, the gradient, and the magnitudes its rounding error is proportional to."""
    n, v = x.shape
    x = x.double()
    m = x.amax(1, keepdim=True)
    none = m == -float("inf")
    t = x - torch.where(none, torch.zeros_like(m), m)
    log_s = torch.log(torch.exp(t).sum(1, keepdim=True))
    lp = torch.where(none, torch.full_like(t, -float("inf")), t - log_s)
    p = torch.exp(lp)
    h = -torch.where(p > 0, p * lp, torch.where(torch.isnan(p), p, torch.zeros_like(p))).sum(1)
    known = (target != ignore) & (target >= 0) & (target < v)
    at = torch.where(known, target, torch.zeros_like(target))
    got = torch.where(known, lp.gather(1, at[:, None])[:, 0], torch.zeros(n, dtype=torch.float64))
    order = torch.where(torch.isnan(x), torch.full_like(x, float("inf")), x)
    idx = torch.sort(torch.where(torch.isnan(x), 1, 0), dim=1, descending=True, stable=True).indices
    idx = idx.gather(1, torch.sort(order.gather(1, idx), dim=1, descending=True, stable=True).indices)
    idx = idx[:, :k]
    out = dict(log_prob=got, entropy=h, top=lp.gather(1, idx), index=idx)
    ls = torch.where(none, torch.zeros_like(log_s), log_s)[:, 0]
    out["size"] = 1 + ls.abs() + torch.where(known & torch.isfinite(got), got.abs(), torch.zeros_like(got))
    out["top_size"] = 1 + ls.abs()[:, None] + torch.where(torch.isfinite(out["top"]), out["top"].abs(), torch.zeros_like(out["top"]))
    out["h_size"] = 1 + ls.abs() + torch.where(p > 0, p * t.abs(), torch.zeros_like(p)).sum(1)
    if g_lp is not None:
        a = torch.where(known, g_lp.double(), torch.zeros_like(got))
        G = a + g_top.double().sum(1)
        gh = g_h.double()[:, None]
        ent = torch.where(p > 0, lp + h[:, None], torch.zeros_like(lp))
        dx = -p * (G[:, None] + gh * ent)
        dx.scatter_add_(1, at[:, None], a[:, None])
        dx.scatter_add_(1, idx, g_top.double())
        out["dx"] = torch.where(none, torch.zeros_like(dx), dx)
        size = p * (a.abs() + g_top.double().abs().sum(1))[:, None] + p * gh.abs() * (ent.abs() + 1 + h[:, None])
        tt = torch.where(p > 0, t.abs(), torch.zeros_like(t))
        gathered = torch.zeros_like(dx).scatter_add_(1, at[:, None], a.abs()[:, None]).scatter_add_(1, idx, g_top.double().abs())
        out["dx_size"] = size * (1 + tt + ls.abs()[:, None]) + gathered
    return out


def check_lp(r, ref, what):
    """A log probability errs by u times the exponent, log S and itself, and by the relative error of S: 48 roundings of
    the sum plus 2 |t| u of each exponential's argument, averaged: under 128 u (1 + log S + |lp|) together."""
    within(r.log_prob, ref["log_prob"], 128 * U * ref["size"], f"{what} log_prob")
    within(r.entropy, ref["entropy"], 256 * U * ref["h_size"], f"{what} entropy")
    assert torch.equal(r.top_indices.cpu(), ref["index"]), what
    within(r.top_log_probs, ref["top"], 128 * U * ref["top_size"], f"{what} top")


def lp_case(n, v, kind, k, seed=0, masked=True, ties=False):
    g = torch.Generator().manual_seed(77 * n + v + seed)
    x = 3 * torch.randn(n, v, generator=g)
    if ties:
        x = torch.round(x)
    if masked and v > 4:
        x[torch.rand(n, v, generator=g) < 0.1] = -float("inf")
    x = x.to(kind)
    t = torch.randint(0, v, (n,), generator=g)
    if n > 2:
        t[1], t[2] = -1, v + 5                  # ignored, and no class at all
    grads = [torch.randn(n, generator=g), 0.3 * torch.randn(n, generator=g), 0.3 * torch.randn(n, k, generator=g)]
    return x, t, grads


LP_ROWS = [(1, 1, 1), (1, 2, 2), (5, 3, 0), (4, 7, 7), (9, 64, 64), (6, 65, 5), (256, 1000, 5), (3, 1000, 64), (2, 2048, 20),
           (2, 2049, 20), (3, 4096, 0), (1, 5000, 64), (3, 50021, 8), (1, 131072, 20), (40, 8193, 3), (1100, 2500, 2), (5121, 20, 3), (1281, 5, 0), (4099, 64, 8), (6401, 100, 9), (8200, 128, 5), (32769, 128, 9),
           (16390, 64, 33), (8300, 129, 1), (70, 1024, 4), (70, 1025, 4), (40, 4096, 9), (40, 4097, 9)]


@gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n,v,k", LP_ROWS)
def test_log_probs_rows(n, v, k, kind):
    from erfnet_pytorch_amd import functional as hipf
    x, t, gr = lp_case(n, v, TYPES[kind], k)
    leaf = x.to(DEV).requires_grad_()
    r = hipf.log_probs(leaf, t.to(DEV), k)
    assert r.log_prob.dtype == r.entropy.dtype == r.top_log_probs.dtype == torch.float32
    ref = lp_reference(x, t, k, -1, *gr)
    check_lp(r, ref, (n, v, k, kind))
    dx, = torch.autograd.grad([r.log_prob, r.entropy, r.top_log_probs], leaf, [g.to(DEV) for g in gr])
    assert dx.dtype == x.dtype
    stored = half_step(x.dtype)
    within(dx, ref["dx"], stored * ref["dx"].abs() + 256 * U * ref["dx_size"] + 1e-36, (n, v, k, kind, "dx"))
    with torch.no_grad():
        for a, b in zip(hipf.log_probs(leaf, t.to(DEV), k), r):
            assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n,v,h,w,k", [(2, 20, 64, 33, 2), (1, 20, 80, 64, 8), (2, 5, 70, 40, 0), (1, 2, 4099, 1, 1),
                                       (1, 256, 64, 65, 4), (2, 20, 5, 7, 3), (1, 257, 65, 64, 3), (2, 40, 64, 64, 12)])
def test_log_probs_of_pixels(n, v, h, w, k, kind):
    """[N,K,H,W] with dim 1, over the pixel kernel's bounds on pixels, classes and alternatives, in NCHW and NHWC memory."""
    from erfnet_pytorch_amd import functional as hipf
    x, t, gr = lp_case(n * h * w, v, TYPES[kind], k, ties=True)
    ref = lp_reference(x, t, k, -1, *gr)
    image = lambda a, c: a.view(n, h, w, c).permute(0, 3, 1, 2).contiguous().to(DEV)      # noqa: E731
    plane = lambda a: a.view(n, h, w).to(DEV)       # noqa: E731
    rows = lambda a: a.permute(0, 2, 3, 1).reshape(n * h * w, -1)       # noqa: E731
    for fmt in (torch.contiguous_format, torch.channels_last):
        leaf = image(x, v).to(memory_format=fmt).requires_grad_()
        r = hipf.log_probs(leaf, plane(t), k, dim=1)
        assert r.top_indices.shape == (n, k, h, w) and r.entropy.shape == (n, h, w)
        flat = hipf.LogProbs(r.log_prob.reshape(-1), r.entropy.reshape(-1), rows(r.top_log_probs), rows(r.top_indices))
        check_lp(flat, ref, (n, v, h, w, k, kind))
        dx, = torch.autograd.grad([r.log_prob, r.entropy, r.top_log_probs], leaf,
                                  [plane(gr[0]), plane(gr[1]), image(gr[2], k)])
        within(rows(dx), ref["dx"], half_step(x.dtype) * ref["dx"].abs() + 256 * U * ref["dx_size"] + 1e-36, "dx")


@gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("v", [40, 1000, 3000, 20000])
def test_log_probs_masked_and_non_finite_rows(v, kind):
    """All classes masked; masks of the type's lowest value; one class left; NaN; +infinity; the lowest value everywhere."""
    from erfnet_pytorch_amd import functional as hipf
    x, t, gr = lp_case(8, v, torch.float32, 4, masked=False)
    low = torch.finfo(TYPES[kind]).min
    x[0] = -float("inf")
    x[1, ::2] = low
    x[2] = -float("inf")
    x[2, v // 2] = 1.5
    x[3] = low
    x[4, 3] = float("nan")
    x[5, 7] = float("inf")
    x[6, :] = 2.0
    t = torch.tensor([1, 2, v // 2, 0, 1, 2, 5, 0])
    x = x.to(TYPES[kind])
    leaf = x.to(DEV).requires_grad_()
    r = hipf.log_probs(leaf, t.to(DEV), 4)
    ref = lp_reference(x, t, 4, -1, *gr)
    # rows 0..3, 6, 7 by the formula; the two spoilt rows are NaN throughout
    ok = [0, 1, 2, 3, 6, 7]
    cut = lambda d: {n: a[ok] for n, a in d.items()}      # noqa: E731
    check_lp(hipf.LogProbs(*(a[ok] for a in r)), cut(ref), (v, kind))
    assert r.entropy[0] == 0 and r.entropy[2] == 0 and r.log_prob[2] == 0
    assert r.top_indices[4, 0] == 3 and r.top_indices[5, 0] == 7
    for o in (r.log_prob, r.entropy, r.top_log_probs):
        assert torch.isnan(o[4:6]).all()
    dx, = torch.autograd.grad([r.log_prob, r.entropy, r.top_log_probs], leaf, [g.to(DEV) for g in gr])
    within(dx[ok], ref["dx"][ok], half_step(x.dtype) * ref["dx"][ok].abs() + 256 * U * ref["dx_size"][ok] + 1e-36, "dx")
    assert torch.equal(dx[0].float().cpu(), torch.zeros(v))
    assert torch.isnan(dx[4]).all()


@gpu
@pytest.mark.parametrize("v", [1000, 30000])
@pytest.mark.parametrize("how", ["rising", "falling", "equal"])
def test_log_probs_alternatives_of_ordered_rows(v, how):
    """Orders that fill the candidate buffer at every step, and rows of ties (the lowest indices win)."""
    from erfnet_pytorch_amd import functional as hipf
    base = torch.arange(v, dtype=torch.float32) / v
    x = {"rising": base, "falling": base.flip(0), "equal": torch.zeros(v)}[how].expand(3, v).contiguous()
    t = torch.zeros(3, dtype=torch.int64)
    r = hipf.log_probs(x.to(DEV), t.to(DEV), 64)
    check_lp(r, lp_reference(x, t, 64, -1), (v, how))


@gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,v", [(1301, 20011), (40_001, 701), (2_600_000, 10)])
def test_log_probs_gradient_of_many_rows_equals_that_of_few(rows, v, kind):
    """Gradients of 48 MB and more take other stores than small ones: the same rows in four calls give them bit for bit."""
    from erfnet_pytorch_amd import functional as hipf
    g = torch.Generator(device=DEV).manual_seed(v)
    x = torch.randn(rows, v, generator=g, device=DEV).to(TYPES[kind])
    t = torch.randint(0, v, (rows,), generator=g, device=DEV)
    gs = [torch.randn(rows, generator=g, device=DEV), torch.randn(rows, 3, generator=g, device=DEV)]
    got = []
    for step in (rows, -(-rows // 4)):
        dx = []
        for a in range(0, rows, step):
            part = x[a:a + step].clone().requires_grad_()
            r = hipf.log_probs(part, t[a:a + step], 3)
            dx += torch.autograd.grad([r.log_prob, r.top_log_probs], part, [u[a:a + step] for u in gs])
        got.append(torch.cat(dx))
    if v == 10:         # (short rows go by another kernel at any count from 2560 on)
        assert torch.equal(got[0], got[1])
        return
    # the statistics of a row depend on how many threads share it, and that on how many rows there are: two of them, rounded
    bound = half_step(x.dtype) * 2 * got[1].double().abs() + 512 * U * (1 + got[1].double().abs())
    assert ((got[0].double() - got[1].double()).abs() <= bound).all()


@gpu
@pytest.mark.parametrize("kind", TYPES)
def test_log_probs_gradient_of_many_pixels_equals_that_of_each_image(kind):
    from erfnet_pytorch_amd import functional as hipf
    n, v, h, w = 7, 20, 256, 739
    g = torch.Generator(device=DEV).manual_seed(5)
    x = torch.randn(n, v, h, w, generator=g, device=DEV).to(TYPES[kind])
    t = torch.randint(0, v, (n, h, w), generator=g, device=DEV)
    gs = [torch.randn(n, h, w, generator=g, device=DEV), torch.randn(n, 2, h, w, generator=g, device=DEV)]
    got = []
    for step in (n, 1):
        dx = []
        for a in range(0, n, step):
            part = x[a:a + step].clone().requires_grad_()
            r = hipf.log_probs(part, t[a:a + step], 2, 1)
            dx += torch.autograd.grad([r.entropy, r.top_log_probs], part, [u[a:a + step] for u in gs])
        got.append(torch.cat(dx))
    assert torch.equal(got[0], got[1])


@gpu
@pytest.mark.parametrize("k", [1, 7, 64])
@pytest.mark.parametrize("v,rows", [(9001, 5), (9001, 1100), (50003, 3), (100003, 2)])
def test_log_probs_alternatives_among_many_ties(v, rows, k):
    """Few distinct values (the lowest indices of the largest win, wherever it begins), masked rows and columns, rows at every
    alignment: a wave a row, a block a row and several blocks a row."""
    from erfnet_pytorch_amd import functional as hipf
    g = torch.Generator().manual_seed(v + k)
    x = torch.randint(0, 3, (5, v), generator=g).float()
    x[1] = -float("inf")
    x[2, : v // 2] = 0.0
    x[3].clamp_(max=1.0)
    x[3, -5:] = 2.0
    x[4, torch.rand(v, generator=g) < 0.5] = -float("inf")
    x = x.repeat(-(-rows // 5), 1)[:rows].contiguous()
    t = torch.randint(0, v, (rows,), generator=g)
    r = hipf.log_probs(x.to(DEV).bfloat16(), t.to(DEV), k)
    ref = lp_reference(x[:5], t[:5], k, -1)
    check_lp(hipf.LogProbs(*(o[:5] for o in r)), ref, (v, rows, k))
    assert torch.equal(r.top_indices[-5:], r.top_indices[:5])       # (rows is below 5 or a multiple of it)


@gpu
def test_log_probs_last_position_of_padded_batch_and_leading_shapes():
    """logits[:, -1] of a [B, S, V] tensor is read in place with a row stride; a 1-D row; expanded rows; no rows."""
    from erfnet_pytorch_amd import functional as hipf
    x, t, gr = lp_case(12, 777, torch.bfloat16, 3)
    full = x.view(3, 4, 777).to(DEV).requires_grad_()
    pick = torch.tensor([3, 7, 11])
    r = hipf.log_probs(full[:, -1], t[pick].to(DEV), 3)
    ref = lp_reference(x[pick], t[pick], 3, -1, *(g[pick] for g in gr))
    check_lp(r, ref, "last position")
    dx, = torch.autograd.grad([r.log_prob, r.entropy, r.top_log_probs], full, [g[pick].to(DEV) for g in gr])
    within(dx[:, -1], ref["dx"], half_step(x.dtype) * ref["dx"].abs() + 256 * U * ref["dx_size"] + 1e-36, "dx")
    assert not dx[:, :-1].any()
    r = hipf.log_probs(x.view(3, 4, 777).to(DEV), t.view(3, 4).to(DEV), 3)
    assert r.log_prob.shape == (3, 4) and r.top_indices.shape == (3, 4, 3)
    check_lp(hipf.LogProbs(r[0].view(-1), r[1].view(-1), r[2].view(-1, 3), r[3].view(-1, 3)), lp_reference(x, t, 3, -1), "3-D")
    one = hipf.log_probs(x[0].to(DEV), t[0].to(DEV), 2)
    assert one.log_prob.shape == () and one.top_indices.shape == (2,)
    wide = hipf.log_probs(x[:1].to(DEV).expand(5, 777), t[:1].to(DEV).expand(5), 2)
    assert torch.equal(wide.log_prob, one.log_prob.expand(5)) and torch.equal(wide.top_indices, one.top_indices.expand(5, 2))
    skip = hipf.log_probs(x.to(DEV)[:, ::2], torch.zeros(12, dtype=torch.int64, device=DEV), 2)
    check_lp(skip, lp_reference(x[:, ::2], torch.zeros(12, dtype=torch.int64), 2, -1), "every other class")
    empty = hipf.log_probs(x.to(DEV)[:0], t.to(DEV)[:0], 2)
    assert empty.log_prob.shape == (0,) and empty.top_indices.shape == (0, 2)


@gpu
def test_log_probs_ignore_index_and_single_gradients():
    from erfnet_pytorch_amd import functional as hipf
    x, t, gr = lp_case(20, 30, torch.float32, 4)
    t = t.clamp(0, 29)
    t[3] = t[9] = 7
    leaf = x.to(DEV).requires_grad_()
    zero = [torch.zeros_like(g) for g in gr]
    for which in range(3):
        r = hipf.log_probs(leaf, t.to(DEV), 4, ignore_index=7)
        only = [gr[i] if i == which else zero[i] for i in range(3)]
        ref = lp_reference(x, t, 4, 7, *only)
        check_lp(r, ref, which)
        dx, = torch.autograd.grad((r.log_prob, r.entropy, r.top_log_probs)[which], leaf, gr[which].to(DEV))
        within(dx, ref["dx"], 256 * U * ref["dx_size"] + 1e-36, (which, "dx"))
    assert r.log_prob[3] == 0 and r.log_prob[9] == 0


@gpu
def test_log_probs_agree_with_cross_entropy():
    """-mean of the labelled pixels' log probabilities is the framework's cross entropy; both gradients agree."""
    from erfnet_pytorch_amd import functional as hipf
    x, t, _ = lp_case(2 * 48 * 64, 20, torch.float32, 0, masked=False)
    t = t.clamp(-1, 19)
    a = x.view(2, 48, 64, 20).permute(0, 3, 1, 2).contiguous().to(DEV).requires_grad_()
    b = a.detach().clone().requires_grad_()
    tg = t.view(2, 48, 64).to(DEV)
    loss = hipf.cross_entropy(a, tg, -1)
    mine = -hipf.log_probs(b, tg, 0, 1).log_prob.sum() / (tg >= 0).sum()
    loss.backward(), mine.backward()
    assert abs(float(loss.detach()) - float(mine.detach())) <= 1e-5 * abs(float(loss.detach()))
    # p / count: both sides' relative error of p is below 256 u (1 + |t| + log S) with |t| < 32, log S < 4
    n = float((tg >= 0).sum())
    assert (a.grad - b.grad).abs().max() <= 2 * 256 * 37 * U / n


@gpu
def test_log_probs_beyond_32_bit_offsets():
    """Rows and pixels whose last elements lie past 2^31, beside the same ones by themselves.  A row's segments depend on how
    many rows there are, so its sums may differ in the last bits: 1e-5 of numbers below 20.  Pixels agree bit for bit."""
    from erfnet_pytorch_amd import functional as hipf
    v, rows = 65537, 32800
    tail, t, _ = lp_case(3, v, torch.bfloat16, 4)
    t = torch.tensor([5, v - 1, 7])
    x = torch.zeros(rows, v, dtype=torch.bfloat16, device=DEV)
    x[-3:] = tail.to(DEV)
    tg = torch.zeros(rows, dtype=torch.int64, device=DEV)
    tg[-3:] = t.to(DEV)
    x.requires_grad_()
    r = hipf.log_probs(x, tg, 4)
    dx, = torch.autograd.grad(r.log_prob, x, torch.ones(rows, device=DEV))
    part = tail.to(DEV).requires_grad_()
    p = hipf.log_probs(part, t.to(DEV), 4)
    dp, = torch.autograd.grad(p.log_prob, part, torch.ones(3, device=DEV))
    assert (r.log_prob[-3:] - p.log_prob).abs().max() <= 2e-4 and torch.equal(r.top_indices[-3:], p.top_indices)
    assert (dx[-3:].float() - dp.float()).abs().max() <= 2.0 ** -8
    del x, dx, r
    k, n = 66, 1 << 25
    x = torch.zeros(1, k, n, dtype=torch.bfloat16, device=DEV)
    x[:, :, -300:] = torch.randn(1, k, 300, generator=torch.Generator().manual_seed(2)).to(DEV)
    tg = torch.full((1, n), 3, dtype=torch.int64, device=DEV)
    x.requires_grad_()
    r = hipf.log_probs(x, tg, 2, dim=1)
    dx, = torch.autograd.grad(r.log_prob, x, torch.ones(1, n, device=DEV))
    part = x.detach()[:, :, -8192:].contiguous().requires_grad_()
    p = hipf.log_probs(part, tg[:, -8192:].contiguous(), 2, dim=1)
    dp, = torch.autograd.grad(p.log_prob, part, torch.ones(1, 8192, device=DEV))
    for a, b in ((r.log_prob[:, -8192:], p.log_prob), (r.entropy[:, -8192:], p.entropy), (dx[:, :, -8192:], dp),
                 (r.top_indices[:, :, -8192:], p.top_indices)):
        assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("op", ["layer_norm", "log_probs"])
def test_deferred_logits_of_the_network(op):
    """net_classification.Net hands out logits whose kernel has not run; these two read the memory itself, so they run it
    first.  Same numbers and parameter gradients as with logits that are written at once."""
    from erfnet_pytorch_amd import functional as hipf, net_classification
    torch.manual_seed(0)
    net = net_classification.Net(softmax_classes=20).to(DEV).train()
    x = torch.rand(1, 3, 64, 128, generator=torch.Generator().manual_seed(1)).to(DEV)
    t = torch.randint(-1, 20, (1, 64, 128), generator=torch.Generator().manual_seed(2)).to(DEV)
    results = []
    for lazy in (False, True):
        old = hipf.set_lazy_logits(lazy)
        try:
            logits = net(x)
            logits = logits[0] if isinstance(logits, (tuple, list)) else logits
            if op == "layer_norm":
                out = hipf.layer_norm(logits, dim=1)
                loss = (out * out * t.unsqueeze(1)).sum()
            else:
                out = hipf.log_probs(logits, t, 2, 1)
                loss = -(out.log_prob + 0.1 * out.entropy).mean()
                out = out.log_prob
            w = net.encoder.initial_block.conv.weight
            results.append((out.detach(), torch.autograd.grad(loss, w)[0]))
        finally:
            hipf.set_lazy_logits(old)
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])
    assert results[0][0].abs().max() > 0 and results[0][1].abs().max() > 0


@gpu
def test_operands_on_two_devices_are_refused():
    from erfnet_pytorch_amd import functional as hipf
    x = torch.zeros(4, 8, device=DEV)
    with pytest.raises(RuntimeError, match="cpu"):
        hipf.log_probs(x, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="cpu"):
        hipf.layer_norm(x, torch.ones(8))


@gpu
@pytest.mark.parametrize("op", ["layer_norm", "log_probs"])
def test_gradients_are_not_differentiable(op):
    from erfnet_pytorch_amd import functional as hipf
    x = torch.randn(4, 32, generator=torch.Generator().manual_seed(1)).to(DEV).requires_grad_()
    y = hipf.layer_norm(x) if op == "layer_norm" else hipf.log_probs(x, torch.zeros(4, dtype=torch.int64, device=DEV)).log_prob
    plain, = torch.autograd.grad((y * y).sum(), x, retain_graph=True)
    dx, = torch.autograd.grad((y * y).sum(), x, create_graph=True)
    assert torch.equal(dx, plain)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(dx.sum(), x)


# ================================================================================ AdamW
HP = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)


def adamw_reference(p, g, m, v, step, hp):
    """One step in float64 from the given state.  The last result is the size that 24 u of the update's error goes by: the
    update with |b1 m| + |(1 - b1) g| in the place of m, whose two terms may cancel while their roundings do not."""
    b1, b2 = hp["betas"]
    p, g = p.double(), g.double()
    size = b1 * m.abs() + (1 - b1) * g.abs()
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    rate = hp["lr"] / (1 - b1 ** step) / (torch.sqrt(v / (1 - b2 ** step)) + hp["eps"])
    return p - hp["lr"] * hp["weight_decay"] * p - rate * m, m, v, rate * size


def adamw_tensors(sizes, kind, seed=0):
    g = torch.Generator().manual_seed(seed)
    ps = [torch.randn(n, generator=g).to(kind) for n in sizes]
    gs = [[(torch.randn(n, generator=g) * torch.exp(torch.randn(n, generator=g))).to(kind) for n in sizes] for _ in range(4)]
    return ps, gs


ADAMW_SIZES = [[1], [255, 256, 257], [4095, 4096, 4097, 3], [8, 0, 5], [10000] + [17 * i + 1 for i in range(120)]]


def decode(st, key, shape):
    codes, scale = st[key].float().flatten().double(), st[key + "_scale"].double()
    return (codes * scale.repeat_interleave(256)[:codes.numel()]).view(shape)


@gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("sizes", ADAMW_SIZES, ids=lambda s: f"{len(s)}x{s[0]}")
def test_adamw_steps(sizes, bits, kind):
    """Every step from the state that the optimiser holds: m to 4 u of its terms, v to 6 u, the parameter to 3 u of
    itself and 24 u of its update (a dozen roundings, the scalars' own among them) plus its own storage; 8-bit
    moments to half a step of e4m3 (2^-4 of the value, 2^-10 of the scale below its least normal number)."""
    from erfnet_pytorch_amd import optim
    ps, gs = adamw_tensors(sizes, TYPES[kind], seed=len(sizes))
    params = [torch.nn.Parameter(p.to(DEV)) for p in ps]
    opt = optim.AdamW(params, **HP, state_bits=bits)
    for step in range(1, 5):
        before = []
        for p, g in zip(params, gs[step - 1]):
            p.grad = g.to(DEV)
            st = opt.state[p]
            if not st:
                m = v = torch.zeros(p.shape, dtype=torch.float64)
            elif bits == 32:
                m, v = st["exp_avg"].double().cpu(), st["exp_avg_sq"].double().cpu()
            else:
                cpu = {k: t.cpu() for k, t in st.items()}
                m, v = decode(cpu, "exp_avg", p.shape), decode(cpu, "exp_avg_sq_root", p.shape) ** 2
            before.append((p.detach().cpu().clone(), m, v))
        opt.step()
        for i, (p, (p0, m0, v0)) in enumerate(zip(params, before)):
            g = gs[step - 1][i]
            ref, m, v, upd = adamw_reference(p0, g, m0, v0, step, HP)
            what = (sizes[i], bits, kind, step)
            within(p.detach(), ref, half_step(p.dtype) * ref.abs() + 3 * U * p0.double().abs() * (1 + half_step(p.dtype)) + 24 * U * upd.abs() * 1.01, what)
            st = {k: t.cpu() for k, t in opt.state[p].items()}
            assert float(st["step"]) == step
            m_tol = 4 * U * (m0.abs() + g.double().abs())
            if bits == 32:
                within(st["exp_avg"], m, m_tol, (what, "m"))
                within(st["exp_avg_sq"], v, 6 * U * v, (what, "v"))
                continue
            for key, x, tol, root in (("exp_avg", m, m_tol, False), ("exp_avg_sq_root", torch.sqrt(v), 8 * U * torch.sqrt(v), True)):
                scale = st[key + "_scale"].double()
                n = x.numel()
                blocks = lambda t: torch.nn.functional.pad(t, (0, -n % 256)).view(-1, 256)       # noqa: E731
                top, top_tol = (blocks(t).amax(1) if n else x.new_zeros(0) for t in (x.abs(), tol))
                # |max |x + e| - max |x|| <= max |e|: the moment's own error enters whole, it is not relative to the
                # largest moment (b1 m and (1 - b1) g may cancel in all of a block's elements); two roundings behind it
                within(st[key + "_scale"], top / 448, (10 * U * top + top_tol) / 448 + 1e-40, (what, key, "scale"))
                s = scale.repeat_interleave(256)[:n]
                half = torch.maximum(x.abs() * 2.0 ** -4, s * 2.0 ** -10) * (1 + 1e-5) + tol
                if root:        # never below the least code
                    half = torch.where((x > 0) & (x < s * 2.0 ** -9), s * 2.0 ** -9 * (1 + 1e-5), half)
                within(decode(st, key, x.shape), x, half, (what, key))
                if root:
                    assert ((x > 1e-20) <= (st[key].float() > 0)).all(), what


@gpu
@pytest.mark.parametrize("wd", [0.0, 0.05])
def test_adamw_follows_torch_and_shares_its_state_dict(wd):
    """Ten steps beside torch.optim.AdamW (fp32): per step both err by a few u of the parameter and its update."""
    from erfnet_pytorch_amd import optim
    sizes = [300, 77, 1, 5000]
    ps, gs = adamw_tensors(sizes, torch.float32, seed=9)
    mine = [torch.nn.Parameter(p.to(DEV)) for p in ps]
    theirs = [torch.nn.Parameter(p.to(DEV)) for p in ps]
    hp = dict(HP, weight_decay=wd)
    a, b = optim.AdamW(mine, **hp), torch.optim.AdamW(theirs, **hp, foreach=False, fused=False)
    for i in range(10):
        if i == 5:              # the state travels both ways
            sa, sb = a.state_dict(), b.state_dict()
            a = optim.AdamW(mine, **hp)
            b = torch.optim.AdamW(theirs, **hp, foreach=False, fused=False)
            a.load_state_dict(sb)
            b.load_state_dict(sa)
        for p, q, g in zip(mine, theirs, gs[i % 4]):
            p.grad, q.grad = g.to(DEV), g.to(DEV)
        a.step(), b.step()
    for p, q in zip(mine, theirs):
        assert (p - q).abs().max() <= 10 * (8 * U * p.abs().max() + 64 * U * HP["lr"] * 10)


@gpu
def test_adamw_takes_the_state_of_torchs_bf16_optimiser():
    """torch.optim.AdamW holds a bf16 parameter's moments in bf16; they are widened, and the next step is the formula's."""
    from erfnet_pytorch_amd import optim
    (p0,), gs = adamw_tensors([500], torch.bfloat16, seed=12)
    theirs = torch.nn.Parameter(p0.to(DEV))
    b = torch.optim.AdamW([theirs], **HP, foreach=False)
    theirs.grad = gs[0][0].to(DEV)
    b.step()
    mine = torch.nn.Parameter(theirs.detach().clone())
    a = optim.AdamW([mine], **HP)
    a.load_state_dict(b.state_dict())
    st = {k: t.cpu() for k, t in a.state[mine].items()}
    assert st["exp_avg"].dtype == st["exp_avg_sq"].dtype == torch.float32
    mine.grad = gs[1][0].to(DEV)
    before = mine.detach().cpu().clone()
    a.step()
    ref, _, _, upd = adamw_reference(before, gs[1][0], st["exp_avg"].double(), st["exp_avg_sq"].double(), 2, HP)
    within(mine.detach(), ref, 2.0 ** -8 * ref.abs() + 4 * U * before.double().abs() + 25 * U * upd, "step 2")


@gpu
def test_adamw8_state_dict_round_trip_and_refusals():
    from erfnet_pytorch_amd import optim
    ps, gs = adamw_tensors([300, 513], torch.bfloat16, seed=4)
    def make(bits=8):
        q = [torch.nn.Parameter(p.to(DEV)) for p in ps]
        return q, optim.AdamW(q, **HP, state_bits=bits)
    a, oa = make()
    for i in range(2):
        for p, g in zip(a, gs[i]):
            p.grad = g.to(DEV)
        oa.step()
    b, ob = make()
    ob.load_state_dict(oa.state_dict())
    with torch.no_grad():
        for p, q in zip(a, b):
            q.copy_(p)
    for p, q, g in zip(a, b, gs[2]):
        p.grad, q.grad = g.to(DEV), g.to(DEV)
    oa.step(), ob.step()
    for p, q in zip(a, b):
        assert torch.equal(p, q)
        for k, t in oa.state[p].items():
            u = ob.state[q][k]
            assert u.dtype == t.dtype and torch.equal(u.float(), t.float()) and (k == "step" or u.data_ptr() != t.data_ptr())
    with pytest.raises(ValueError, match="state_bits"):
        make(32)[1].load_state_dict(oa.state_dict())


@gpu
def test_adamw8_special_values():
    """Zero blocks stay zero; NaN and infinity stay in their own element; a tiny block is stored as zeros; an element
    whose root would round to zero keeps the least code, so that its step stays bounded when its gradient stops."""
    from erfnet_pytorch_amd import optim
    p = torch.nn.Parameter(torch.ones(5 * 256, device=DEV))
    opt = optim.AdamW([p], lr=1e-3, weight_decay=0.0, state_bits=8)
    g = torch.zeros(5, 256)
    g[1] = 1.0
    g[1, 3], g[1, 200] = float("nan"), float("inf")
    g[2] = 1e-37
    g[3] = 1.0
    g[3, 5] = 1e-9
    p.grad = g.view(-1).to(DEV)
    opt.step()
    st = opt.state[p]
    m, r = st["exp_avg"].float().view(5, 256).cpu(), st["exp_avg_sq_root"].float().view(5, 256).cpu()
    for t, s in ((m, st["exp_avg_scale"]), (r, st["exp_avg_sq_root_scale"])):
        assert s[0] == 0 and not t[0].any() and not t[4].any()
        assert torch.isnan(t[1, [3, 200]]).all() and torch.equal(torch.isnan(t).sum(1), torch.tensor([0, 2, 0, 0, 0]))
        assert (t[1, :3] == 448).all()
    assert not m[2].any() and st["exp_avg_scale"][2] == 0
    assert r[3, 5] == 2.0 ** -9
    x = p.detach().view(5, 256).cpu()
    assert torch.isnan(x[1, [3]]).all() and torch.isfinite(x[[0, 2, 3, 4]]).all() and (x[0] == 1).all()
    before = p.detach().clone()
    p.grad = torch.zeros_like(p)
    opt.step()
    moved = (p.detach() - before).view(5, 256)[3].abs()
    assert moved.max() <= 2e-3, float(moved.max())


@gpu
def test_adamw_groups_schedules_missing_gradients_and_flat_parameters():
    from erfnet_pytorch_amd import optim
    ps, gs = adamw_tensors([40, 300, 50], torch.float32, seed=2)
    params = [torch.nn.Parameter(p.to(DEV)) for p in ps]
    opt = optim.AdamW([dict(params=params[:2], lr=1e-2), dict(params=params[2:], weight_decay=0.5)], **HP)
    m = [torch.zeros(p.shape, dtype=torch.float64) for p in ps]
    v = [torch.zeros(p.shape, dtype=torch.float64) for p in ps]
    ref = [p.double() for p in ps]
    steps = [0, 0, 0]
    for i in range(4):
        for j, p in enumerate(params):
            p.grad = None if (j, i) in ((0, 0), (1, 2)) else gs[i][j].to(DEV)
        opt.param_groups[0]["lr"] = 1e-2 / (i + 1)
        opt.step()
        for j, p in enumerate(params):
            if p.grad is None:
                continue
            steps[j] += 1
            hp = dict(HP, lr=1e-2 / (i + 1)) if j < 2 else dict(HP, weight_decay=0.5)
            ref[j], m[j], v[j], _ = adamw_reference(ref[j], gs[i][j], m[j], v[j], steps[j], hp)
    for j, p in enumerate(params):
        assert float(opt.state[p]["step"]) == steps[j]
        # four steps, each a few u of the parameter and 24 u of an update of at most 10 lr
        within(p.detach(), ref[j], 4 * (4 * U * ref[j].abs() + 24 * U * 0.1), j)


@gpu
@pytest.mark.parametrize("kind", TYPES)
def test_adamw_on_a_flat_buffer_equals_its_tensors(kind):
    from erfnet_pytorch_amd import optim
    ps, gs = adamw_tensors([40, 300, 1, 5000], TYPES[kind], seed=8)
    flat = torch.nn.Parameter(torch.cat(ps).to(DEV))
    params = [torch.nn.Parameter(p.to(DEV)) for p in ps]
    a, b = optim.AdamW([flat], **HP), optim.AdamW(params, **HP)
    for i in range(3):
        flat.grad = torch.cat(gs[i]).to(DEV)
        for p, g in zip(params, gs[i]):
            p.grad = g.to(DEV)
        a.step(), b.step()
    assert torch.equal(flat.detach(), torch.cat([p.detach() for p in params]))


@gpu
def test_adamw_views_at_odd_offsets():
    """Parameters, gradients and moments that start at any element of a larger buffer, and what lies behind them stays."""
    from erfnet_pytorch_amd import optim
    for bits in (32, 8):
        base = torch.randn(2000, generator=torch.Generator().manual_seed(1)).to(DEV)
        keep = base.clone()
        p = torch.nn.Parameter(base[3:1003])
        g = torch.randn(1500, generator=torch.Generator().manual_seed(2)).to(DEV)
        p.grad = g[1:1001]
        q = torch.nn.Parameter(base[3:1003].clone())
        q.grad = g[1:1001].clone()
        a, b = optim.AdamW([p], **HP, state_bits=bits), optim.AdamW([q], **HP, state_bits=bits)
        a.step(), b.step()
        assert torch.equal(p, q) and torch.equal(base[:3], keep[:3]) and torch.equal(base[1003:], keep[1003:])


@gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("kind", TYPES)
def test_adamw_of_large_tensors_at_odd_offsets_equals_its_pieces(kind, bits):
    """Tensors of 320 MB and more take other loads and stores than small ones: one step of a large tensor that begins at no
    multiple of a vector is, bit for bit, the steps of its 256-element-aligned pieces."""
    from erfnet_pytorch_amd import optim
    n, piece = 70_000_001, 17_500_160
    g = torch.Generator(device=DEV).manual_seed(3)
    base, grad = (torch.randn(n + 3, generator=g, device=DEV).to(TYPES[kind]) for _ in range(2))
    whole = torch.nn.Parameter(base.clone()[1:n + 1])
    parts = [torch.nn.Parameter(base[1 + a:1 + min(a + piece, n)].clone()) for a in range(0, n, piece)]
    results = []
    for params in ([whole], parts):
        opt = optim.AdamW(params, **HP, state_bits=bits)
        per_launch = [opt] if params is not parts else [optim.AdamW([p], **HP, state_bits=bits) for p in parts]
        for step in range(2):
            at = 3
            for p in params:
                p.grad = grad[at:at + p.numel()]
                at += p.numel()
            for o in per_launch:
                o.step()
        states = [o.state[p] for o in per_launch for p in o.param_groups[0]["params"]]
        results.append([torch.cat([p.detach() for p in params])] +
                       [torch.cat([s[k].view(torch.uint8).flatten() if s[k].dtype == torch.float8_e4m3fn else s[k] for s in states])
                        for k in opt._moments])
    for a, b in zip(*results):
        assert torch.equal(a, b)


@gpu
def test_adamw_refuses_parameters_that_share_memory():
    from erfnet_pytorch_amd import optim
    buf = torch.zeros(100, device=DEV)
    apart = [torch.nn.Parameter(buf[:40]), torch.nn.Parameter(buf[40:]), torch.nn.Parameter(buf[:0])]
    optim.AdamW(apart)
    shared = apart + [torch.nn.Parameter(buf[39:41])]
    with pytest.raises(ValueError, match="share memory"):
        optim.AdamW(shared)
    late = [torch.nn.Parameter(torch.zeros(4)), torch.nn.Parameter(torch.zeros(4))]
    opt = optim.AdamW(late)
    for p in late:
        p.data = buf[:4]
        p.grad = torch.ones(4, device=DEV)
    with pytest.raises(ValueError, match="share memory"):
        opt.step()
    assert not opt.state and not buf.any()


@gpu
def test_adamw_moves_the_version_of_what_it_updates():
    """Copies kept of a parameter go by its version: a bf16 parameter's fp32 copy is fresh after a step."""
    from erfnet_pytorch_amd import functional as hipf, optim
    w = torch.nn.Parameter(torch.ones(64, dtype=torch.bfloat16, device=DEV))
    x = torch.randn(8, 64, generator=torch.Generator().manual_seed(0)).to(DEV)
    first = hipf.layer_norm(x, w).detach()
    opt = optim.AdamW([w], lr=0.5, weight_decay=0.0)
    w.grad = torch.ones_like(w)
    before = w._version
    opt.step()
    assert w._version > before
    assert torch.equal(w.detach().float(), torch.full((64,), 0.5, device=DEV))
    assert torch.equal(hipf.layer_norm(x, w).detach(), first * 0.5)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_copies_and_refuses_capture(bits):
    import copy
    from erfnet_pytorch_amd import optim
    p = torch.nn.Parameter(torch.ones(300, device=DEV))
    opt = optim.AdamW([p], state_bits=bits)
    p.grad = torch.ones_like(p)
    opt.step()
    twin = copy.deepcopy(opt)
    q = twin.param_groups[0]["params"][0]
    q.grad = torch.ones_like(q)
    opt.step(), twin.step()
    assert twin.state_bits == bits and torch.equal(p, q)
    kept = p.detach().clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="captured"):
            opt.step()
        mark = kept * 2
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(p.detach(), kept) and torch.equal(mark, kept * 2) and float(opt.state[p]["step"]) == 2


@gpu
def test_adamw_refuses_state_and_gradients_that_do_not_fit():
    from erfnet_pytorch_amd import optim
    p = torch.nn.Parameter(torch.ones(300, device=DEV))
    opt = optim.AdamW([p], state_bits=8)
    p.grad = torch.ones_like(p)
    opt.step()
    kept = p.detach().clone()
    st = opt.state[p]
    for key, bad, error in (("exp_avg_scale", torch.zeros(1, device=DEV), ValueError),
                            ("exp_avg", torch.zeros(300, device=DEV), ValueError),
                            ("exp_avg_sq_root", torch.zeros(300, dtype=torch.float8_e4m3fn), RuntimeError),
                            ("step", torch.zeros(1, device=DEV), ValueError)):
        good, st[key] = st[key], bad
        with pytest.raises(error):
            opt.step()
        st[key] = good
    st.pop("exp_avg")
    with pytest.raises(KeyError):
        opt.step()
    wide = torch.zeros(300, 2, device=DEV)
    q = torch.nn.Parameter(wide[:, 0])
    q.grad = torch.ones(300, device=DEV)
    with pytest.raises(ValueError, match="contiguous"):
        optim.AdamW([q]).step()
    h = torch.nn.Parameter(torch.ones(4, device=DEV, dtype=torch.float16))
    h.grad = torch.ones_like(h)
    with pytest.raises(TypeError):
        optim.AdamW([h]).step()
    torch.cuda.synchronize()
    assert torch.equal(p.detach(), kept)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_beyond_32_bit_offsets(bits):
    """2^31 + 700 bf16 parameters: the last blocks equal the same elements as a tensor of their own, bit for bit."""
    from erfnet_pytorch_amd import optim
    n, tail = (1 << 31) + 700, 1024 + 188
    g = torch.Generator().manual_seed(6)
    small, grad = torch.randn(tail, generator=g).bfloat16().to(DEV), torch.randn(tail, generator=g).bfloat16().to(DEV)
    p = torch.nn.Parameter(torch.zeros(n, dtype=torch.bfloat16, device=DEV))
    p.grad = torch.zeros_like(p)
    with torch.no_grad():
        p[-tail:] = small
    p.grad[-tail:] = grad
    q = torch.nn.Parameter(small.clone())
    q.grad = grad.clone()
    assert (n - tail) % 256 == 0
    a, b = optim.AdamW([p], **HP, state_bits=bits), optim.AdamW([q], **HP, state_bits=bits)
    for _ in range(2):
        a.step(), b.step()
    assert torch.equal(p.detach()[-tail:], q.detach())
    for key, t in b.state[q].items():
        if key != "step":
            assert torch.equal(a.state[p][key][-t.numel():].view(torch.uint8), t.view(torch.uint8)), key


# ================================================================================ together, streams, graphs
def head_step(hipf, x, w, b, lin, t):
    """Norm, a linear head, log probabilities and an entropy bonus: the loss of one step."""
    r = hipf.log_probs(hipf.layer_norm(x, w, b) @ lin, t, 3)
    return -(r.log_prob.sum() + 0.1 * r.entropy.sum()) / t.numel(), r


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_training_steps_with_all_three(bits):
    """Three steps of a classifier head (norm - linear - log probabilities - AdamW) beside the same in float64 from the
    same parameters each step: every parameter's gradient to 1e-4 of its largest (sums over 64 rows of products of
    a dozen roundings each, and torch's own fp32 matrix product between them)."""
    from erfnet_pytorch_amd import functional as hipf, optim
    g = torch.Generator().manual_seed(11)
    x = torch.randn(64, 32, generator=g)
    t = torch.randint(0, 50, (64,), generator=g)
    params = [torch.nn.Parameter(p.to(DEV)) for p in (torch.ones(32), torch.zeros(32), 0.3 * torch.randn(32, 50, generator=g))]
    opt = optim.AdamW(params, lr=1e-2, state_bits=bits)
    for _ in range(3):
        opt.zero_grad()
        loss, _ = head_step(hipf, x.to(DEV), *params, t.to(DEV))
        loss.backward()
        ref = [p.detach().double().cpu().requires_grad_() for p in params]
        h = torch.nn.functional.layer_norm(x.double(), (32,), ref[0], ref[1], 1e-5) @ ref[2]
        lp = torch.log_softmax(h, 1)
        want = -(lp.gather(1, t[:, None]).sum() - 0.1 * (lp.exp() * lp).sum()) / 64
        want.backward()
        assert abs(float(loss.detach()) - float(want.detach())) <= 1e-5 * abs(float(want.detach()))
        for p, q in zip(params, ref):
            assert (p.grad.double().cpu() - q.grad).abs().max() <= 1e-4 * q.grad.abs().max()
        opt.step()


@gpu
def test_norm_and_log_probs_on_another_stream_and_in_a_graph():
    """The same numbers on a side stream; captured with the backward pass and replayed with new inputs, eager work in
    between; two graphs captured on one stream do not share scratch memory."""
    from erfnet_pytorch_amd import functional as hipf
    g = torch.Generator().manual_seed(5)
    w, b = (t.to(DEV) for t in (1 + 0.1 * torch.randn(5000, generator=g), 0.1 * torch.randn(5000, generator=g)))
    xs = [torch.randn(3, 5000, generator=g).to(DEV) for _ in range(4)]
    t = torch.tensor([5, -1, 4999], device=DEV)
    up = [torch.randn(n, generator=g).to(DEV) for n in ((3,), (3,), (3, 3))]

    def work(x, wl, bl):
        # the framework's own kernels only (a captured library product or sum may record memory-set nodes)
        r = hipf.log_probs(hipf.layer_norm(x, wl, bl), t, 3)
        dw, db = torch.autograd.grad([r.log_prob, r.entropy, r.top_log_probs], (wl, bl), up)
        return [r.log_prob.detach(), r.entropy.detach(), r.top_indices, dw, db]

    def leaves():
        return w.detach().clone().requires_grad_(), b.detach().clone().requires_grad_()
    eager = [work(x, *leaves()) for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = work(xs[0], *leaves())
    side.synchronize()
    for a, c in zip(other, eager[0]):
        assert torch.equal(a, c)
    graphs = []
    del other
    for _ in range(2):
        static = xs[0].clone()
        wl, bl = leaves()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            work(static, wl, bl)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = work(static, wl, bl)
        graphs.append((graph, static, out, wl, bl))       # (the graph reads the leaves' memory: they have to live as long)
    for i in (1, 2, 3, 0):
        for k, (graph, static, out, _, _) in enumerate(graphs):
            static.copy_(xs[(i + k) % 4])
            graph.replay()
        work(xs[0], *leaves())
        torch.cuda.synchronize()
        for k, (graph, static, out, _, _) in enumerate(graphs):
            for a, c in zip(out, eager[(i + k) % 4]):
                assert torch.equal(a, c), (i, k)


# ================================================================================ refusals (no GPU needed)
def test_layer_norm_refusals():
    from erfnet_pytorch_amd import functional as hipf
    x = torch.zeros(4, 8)
    with pytest.raises(RuntimeError, match="GPU"):
        hipf.layer_norm(x)
    with pytest.raises(TypeError, match="fp32 or bf16"):
        hipf.layer_norm(x.half())
    with pytest.raises(ValueError, match="weight shape"):
        hipf.layer_norm(x, torch.ones(7))
    with pytest.raises(ValueError, match="bias shape"):
        hipf.layer_norm(x, None, torch.ones(8, 1))
    with pytest.raises(ValueError, match="dim"):
        hipf.layer_norm(x, dim=0)
    with pytest.raises(ValueError, match="dim"):
        hipf.layer_norm(torch.zeros(()), dim=-1)
    with pytest.raises(ValueError, match="channels"):
        hipf.layer_norm(torch.zeros(2, 16385))
    with pytest.raises(ValueError, match="channels"):
        hipf.layer_norm(torch.zeros(2, 0))
    with pytest.raises(ValueError, match="eps"):
        hipf.layer_norm(x, eps=-1.0)
    with pytest.raises(ValueError, match="eps"):
        hipf.layer_norm(x, eps=float("nan"))


def test_log_probs_refusals():
    from erfnet_pytorch_amd import functional as hipf
    x, t = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="GPU"):
        hipf.log_probs(x, t)
    with pytest.raises(TypeError, match="fp32 or bf16"):
        hipf.log_probs(x.double(), t)
    with pytest.raises(TypeError, match="int64"):
        hipf.log_probs(x, t.int())
    with pytest.raises(ValueError, match="target shape"):
        hipf.log_probs(x, t[:3])
    for k in (-1, 9):
        with pytest.raises(ValueError, match="top_k"):
            hipf.log_probs(x, t, k)
    with pytest.raises(ValueError, match="top_k"):
        hipf.log_probs(torch.zeros(4, 100), t, 65)
    with pytest.raises(ValueError, match="dim"):
        hipf.log_probs(x, t, dim=2)
    with pytest.raises(ValueError, match="classes"):
        hipf.log_probs(torch.zeros(4, 0), t)


def test_adamw_refusals():
    from erfnet_pytorch_amd import optim
    p = torch.nn.Parameter(torch.zeros(4))
    for bad in (dict(lr=-1.0), dict(eps=-1.0), dict(weight_decay=-0.1), dict(betas=(1.0, 0.9)), dict(state_bits=16)):
        with pytest.raises(ValueError):
            optim.AdamW([p], **bad)
    with pytest.raises(ValueError, match="twice"):
        optim.AdamW([p, p])
    with pytest.raises(ValueError, match="twice"):
        optim.AdamW([("a", p), ("b", p)])
    opt = optim.AdamW(iter([p]))
    p.grad = torch.ones(4)
    with pytest.raises(RuntimeError, match="GPU"):
        opt.step()
    opt.param_groups[0]["amsgrad"] = True
    with pytest.raises(NotImplementedError):
        opt.step()


def test_c_entry_points_reject_before_any_launch():
    """Every refusal is decided on the host: these calls return 1 with a message and touch no device."""
    from erfnet_pytorch_amd import _lib
    lib = _lib.lib()
    buf = (C.c_char * 4096)()
    p = C.cast(buf, C.c_void_p)

    def refused(rc, text):
        assert rc != 0
        assert text in lib.erf_last_error().decode(), lib.erf_last_error()
    for name in ("erf_layer_norm_forward", "erf_layer_norm_forward_bf16"):
        f = getattr(lib, name)
        refused(f(p, None, None, p, None, None, 4, 0, 1e-5, None), "channels")
        refused(f(p, None, None, p, None, None, 4, 16385, 1e-5, None), "channels")
        refused(f(p, None, None, p, None, None, -1, 8, 1e-5, None), "row count")
        refused(f(p, None, None, p, None, None, 4, 8, -1.0, None), "eps")
        refused(f(None, None, None, p, None, None, 4, 8, 1e-5, None), "null")
        refused(f(p, None, None, p, p, None, 4, 8, 1e-5, None), "together")
        assert f(p, None, None, p, None, None, 0, 8, 1e-5, None) == 0
    for name in ("erf_layer_norm_backward", "erf_layer_norm_backward_bf16"):
        f = getattr(lib, name)
        refused(f(p, None, p, p, p, p, p, None, 4, 8, None, 0, None), "workspace")
        refused(f(p, None, p, p, p, p, p, None, 4, 8, p, 4, None), "workspace")
        refused(f(p, None, None, p, p, p, None, None, 4, 8, None, 0, None), "null")
    for name in ("erf_log_probs_forward", "erf_log_probs_forward_bf16"):
        f = getattr(lib, name)
        def call(outer=2, v=8, inner=1, ld=8, k=0, top=None, ws=None, n=0, x=p):
            return f(x, p, p, p, p, top, top, outer, v, inner, ld, k, -1, ws, n, None)
        refused(call(v=0), "classes")
        refused(call(v=(1 << 30) + 1), "classes")
        refused(call(outer=-1), "extent")
        refused(call(inner=0), "extent")
        refused(call(k=9, top=p), "top_k")
        refused(call(v=100, ld=100, k=65, top=p), "top_k")
        refused(call(v=100, inner=4, k=9, top=p), "top_k")
        refused(call(k=2), "null")
        refused(call(x=None), "null")
        refused(call(ld=7), "overlap")
        refused(call(outer=1, v=100000, ld=100000), "workspace")
        refused(call(outer=1 << 41), "too many rows")
        refused(call(outer=1 << 40), "too many rows")
        assert call(outer=0) == 0
    for name in ("erf_log_probs_backward", "erf_log_probs_backward_bf16"):
        f = getattr(lib, name)
        refused(f(p, p, p, p, None, p, None, None, p, 2, 8, 1, 8, 2, -1, None), "null")
        refused(f(p, p, p, p, None, p, None, None, p, 2, 0, 1, 8, 0, -1, None), "classes")
    one = (C.c_void_p * 1)(p)
    n = (C.c_longlong * 1)(4)
    for name, tables in (("erf_adamw_step", 4), ("erf_adamw_step_bf16", 4), ("erf_adamw8_step", 6), ("erf_adamw8_step_bf16", 6)):
        f = getattr(lib, name)
        hp = [1e-3, 0.9, 0.999, 1e-8, 0.01]
        refused(f(1, *[one] * tables, n, *hp, 0, None), "step")
        refused(f(-1, *[one] * tables, n, *hp, 1, None), "count")
        refused(f(1, *[one] * tables, n, -1.0, *hp[1:], 1, None), "negative")
        refused(f(1, *[one] * tables, n, hp[0], 1.0, *hp[2:], 1, None), "betas")
        refused(f(1, *[one] * (tables - 1), None, n, *hp, 1, None), "null pointer table")
        refused(f(1, *[one] * (tables - 1), (C.c_void_p * 1)(), n, *hp, 1, None), "null pointer")
        refused(f(1, *[one] * tables, (C.c_longlong * 1)(-1), *hp, 1, None), "negative size")
        assert f(1, *[one] * tables, (C.c_longlong * 1)(0), *hp, 1, None) == 0
