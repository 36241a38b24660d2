"""Layer norm, token log probabilities and AdamW: calls off the ordinary path (other derivatives, tracing, threads, very many
rows, state that arrives late), and bounds that leave no entry of a large result unchecked.  The formulas' references and
the bounds' reasoning are those of test_train_ops.py."""
import pytest
import torch

DEV = "cuda:0"
gpu = pytest.mark.gpu


def noise(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


# ================================================================================ derivatives
def _norm_of(layout):
    """x (a leaf) and y = layer_norm of a layout of it that the kernels read as it is, as a view, or as a copy."""
    from erfnet_pytorch_amd import functional as hipf
    if layout == "rows":
        x = noise(6, 32)
        return x, lambda t: hipf.layer_norm(t)
    if layout == "transposed":
        return noise(32, 6), lambda t: hipf.layer_norm(t.t())
    if layout == "every other row":
        return noise(12, 32), lambda t: hipf.layer_norm(t[::2])
    if layout == "nchw":
        return noise(2, 16, 3, 5), lambda t: hipf.layer_norm(t, dim=1)
    assert layout == "nhwc"
    return noise(2, 16, 3, 5).to(memory_format=torch.channels_last), lambda t: hipf.layer_norm(t, dim=1)


def _logp_of(layout):
    from erfnet_pytorch_amd import functional as hipf
    shape, dim = {"rows": ((6, 32), -1), "tokens": ((2, 3, 32), -1), "one row": ((32,), 0), "moved axis": ((32, 6), 0),
                  "pixels": ((2, 16, 3, 5), 1), "many classes": ((2, 80, 3, 5), 1)}[layout]
    t = torch.zeros(shape[:dim] + shape[dim + 1:] if dim >= 0 else shape[:-1], dtype=torch.int64)
    return noise(*shape), lambda x: hipf.log_probs(x, t.to(DEV), top_k=2, dim=dim)


NORM_LAYOUTS = ["rows", "transposed", "every other row", "nchw", "nhwc"]
LOGP_LAYOUTS = ["rows", "tokens", "one row", "moved axis", "pixels", "many classes"]


def _second(f, x, out, extra):
    """autograd.grad of the gradient, with an upstream gradient that is a constant: only the operator's inputs lead back."""
    x = x.to(DEV).requires_grad_()
    y = out(f(x))
    dx, = torch.autograd.grad(y, x, torch.ones_like(y), create_graph=True)
    if extra:
        dx = dx + x * x
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(dx, x, torch.ones_like(dx), allow_unused=True)


@gpu
@pytest.mark.parametrize("extra", [False, True])
@pytest.mark.parametrize("layout", NORM_LAYOUTS)
def test_second_derivative_of_layer_norm_raises_for_every_layout(layout, extra):
    x, f = _norm_of(layout)
    _second(f, x, lambda y: y, extra)


@gpu
@pytest.mark.parametrize("extra", [False, True])
@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("layout", LOGP_LAYOUTS)
def test_second_derivative_of_log_probs_raises_for_every_layout(layout, which, extra):
    x, f = _logp_of(layout)
    _second(f, x, lambda r: r[which], extra)


@gpu
def test_second_derivative_by_way_of_the_weight_raises():
    from erfnet_pytorch_amd import functional as hipf
    x, w = noise(2, 3, 16).to(DEV).requires_grad_(), noise(16, seed=1).to(DEV).requires_grad_()
    y = hipf.layer_norm(x.transpose(0, 1), w)
    dw, = torch.autograd.grad(y, w, torch.ones_like(y), create_graph=True)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(dw.sum(), x, allow_unused=True)


@gpu
@pytest.mark.parametrize("leaf", [False, True])
@pytest.mark.parametrize("which", ["x", "weight", "bias", "logits"])
def test_forward_mode_raises(which, leaf):
    import torch.autograd.forward_ad as fwd
    from erfnet_pytorch_amd import functional as hipf
    t = {"x": noise(4, 16), "weight": noise(16, seed=1), "bias": noise(16, seed=2), "logits": noise(4, 16)}
    t = {k: v.to(DEV).requires_grad_(leaf) for k, v in t.items()}
    target = torch.zeros(4, dtype=torch.int64, device=DEV)
    with fwd.dual_level():
        t[which] = fwd.make_dual(t[which], torch.ones_like(t[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            if which == "logits":
                hipf.log_probs(t["logits"], target)
            else:
                hipf.layer_norm(t["x"], t["weight"], t["bias"])
    hipf.log_probs(t["logits"].detach(), target)


@gpu
@pytest.mark.parametrize("op", ["layer_norm", "log_probs"])
def test_forward_mode_over_the_gradient_raises(op):
    import torch.autograd.forward_ad as fwd
    from erfnet_pytorch_amd import functional as hipf
    x = noise(4, 16).to(DEV).requires_grad_()
    y = hipf.layer_norm(x) if op == "layer_norm" else hipf.log_probs(x, torch.zeros(4, dtype=torch.int64, device=DEV)).entropy
    with fwd.dual_level():
        g = fwd.make_dual(torch.ones_like(y), torch.ones_like(y))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(y, x, g)


# ================================================================================ tracing
@gpu
@pytest.mark.parametrize("how", ["jit", "fx"])
@pytest.mark.parametrize("op", ["layer_norm", "log_probs"])
def test_tracing_raises(op, how):
    """The results would be constants of the graph: the answer for the example's input, whatever comes."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from erfnet_pytorch_amd import functional as hipf
    x, target = noise(4, 16).to(DEV), torch.zeros(4, dtype=torch.int64, device=DEV)

    def f(t):
        return hipf.layer_norm(t) if op == "layer_norm" else hipf.log_probs(t, target).log_prob

    with pytest.raises(NotImplementedError, match="cannot be traced"):
        torch.jit.trace(f, x) if how == "jit" else make_fx(f)(x)
    f(x)


# ================================================================================ values
@gpu
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("c", [3, 5, 20, 100, 1001, 1030, 5000, 12001, 12004])
def test_layer_norm_gradient_of_high_rows_does_not_overflow_behind_their_end(c, kind):
    """x = 2^113 everywhere: every partial sum is a multiple of it below 2^24 of them, so mean = x and xhat = 0 exactly, and
    dx = (g w - mean(g w)) / sqrt(eps), dw = 0.  mean / sqrt(eps) = 2^113 1e5 is beyond fp32: it must not turn up where a
    vector or a wave reaches beyond the row.  Errors: eps in fp32, root and product (under 8 u), the mean of g w (64 u of the
    mean magnitude), dx's own rounding."""
    from erfnet_pytorch_amd import functional as hipf
    u, rows, eps = 2.0 ** -24, 5, 1e-10
    g, w = noise(rows, c, seed=c, dtype=kind), 1 + 0.3 * noise(c, seed=c + 1)
    x = torch.full((rows, c), 2.0 ** 113, dtype=kind).to(DEV).requires_grad_()
    wd = w.to(DEV).requires_grad_()
    dx, dw = torch.autograd.grad(hipf.layer_norm(x, wd, eps=eps), (x, wd), g.to(DEV))
    gw = g.double() * w.double()
    ref = (gw - gw.mean(1, keepdim=True)) / eps ** 0.5
    size = (gw.abs() + gw.abs().mean(1, keepdim=True)) / eps ** 0.5
    own = 0.0 if kind == torch.float32 else 2.0 ** -8
    off = (dx.cpu().double() - ref).abs() - (72 * u * size * (1 + own) + own * ref.abs())
    assert torch.isfinite(dx).all() and float(off.max()) <= 0
    assert not dw.any()


@gpu
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("c", [20, 1001, 5000, 12001])
def test_layer_norm_of_a_row_whose_spread_is_beyond_fp32(c, kind):
    """One entry of the type's lowest value: the squares sum to infinity, 1 / sqrt(var + eps) is 0, so y = bias and dx = 0, for
    gradients whose product with the row is beyond fp32 too.  The other rows do not notice."""
    from erfnet_pytorch_amd import functional as hipf
    x, g, b = noise(4, c, seed=c, dtype=kind), 30 * noise(4, c, seed=c + 1, dtype=kind), noise(c, seed=c + 2)
    plain = [t.to(DEV).requires_grad_() for t in (x, b)]
    x = x.clone()
    x[1, 3] = torch.finfo(kind).min
    marked = [t.to(DEV).requires_grad_() for t in (x, b)]
    (y0, (dx0, _)), (y, (dx, db)) = (
        (y, torch.autograd.grad(y, t, g.to(DEV))) for t in (plain, marked) for y in [hipf.layer_norm(t[0], None, t[1])])
    assert torch.equal(y[1], b.to(DEV).to(kind)) and not dx[1].any()
    others = [0, 2, 3]
    assert torch.equal(y[others], y0[others]) and torch.equal(dx[others], dx0[others])
    assert torch.isfinite(db).all()


@gpu
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("c", [1, 3, 13, 100, 1000, 1030, 8192, 12000, 16384])
def test_layer_norm_of_constant_rows_is_the_bias(c, kind):
    """Equal values, whose sum fp32 has to round: the differences from the first mean are all the same few units in the last
    place, k of them, so their sum and the sum of their squares are exact below 2^24 units (c k^2), and what is left is zero."""
    from erfnet_pytorch_amd import functional as hipf
    levels = torch.tensor([0.1, 10.3, -1000.1, 1.7, 3.3e-7, 1.1e7, 0.0, 1e30])
    x = levels[:, None].repeat(1, c).to(kind).to(DEV).requires_grad_()
    w, b = noise(c, seed=1).to(DEV).requires_grad_(), noise(c, seed=2).to(DEV).requires_grad_()
    y = hipf.layer_norm(x, w, b)
    assert torch.equal(y, b.to(kind).expand_as(y))
    g = noise(len(levels), c, seed=3, dtype=kind).to(DEV)
    dx, dw = torch.autograd.grad(y, (x, w), g)
    assert not dw.any()                                     # mean = x: xhat is zero in backward too
    # rstd = 1 / sqrt(eps): eps in fp32, root, products (8 u); mean of g w: 64 u of its magnitudes
    gw = g.double() * w.detach().double()
    root = 1e-5 ** -0.5
    ref, size = (gw - gw.mean(1, keepdim=True)) * root, (gw.abs() + gw.abs().mean(1, keepdim=True)) * root
    own = 0.0 if kind == torch.float32 else 2.0 ** -8
    assert float(((dx.double() - ref).abs() - 72 * 2.0 ** -24 * size * (1 + own) - own * ref.abs()).max()) <= 0


@gpu
@pytest.mark.parametrize("c", [100, 1000, 8192, 12000])
def test_layer_norm_error_goes_with_the_spread_and_not_with_the_level(c):
    """Level 1000, spread 0.01.  The differences from the first mean are exact (neighbouring floats), and that mean is off by at
    most 48 u 1000 = 0.3 spreads.  What is left of the differences' mean errs by 64 u of their mean magnitude (below 1.3
    spreads), the variance by 64 u (1 + 0.3^2) of itself, xhat by half of that and a few roundings of its own."""
    from erfnet_pytorch_amd import functional as hipf
    u = 2.0 ** -24
    x, w, b = 1000 + 0.01 * noise(50, c, seed=c), 1 + 0.3 * noise(c, seed=1), 0.3 * noise(c, seed=2)
    y = hipf.layer_norm(*(t.to(DEV) for t in (x, w, b)), eps=1e-12).cpu().double()
    d = x.double() - x.double().mean(1, keepdim=True)
    h = d / torch.sqrt((d * d).mean(1, keepdim=True) + 1e-12)
    ref = h * w.double() + b.double()
    bound = u * (w.double().abs() * (1.3 * 64 + h.abs() * (1.1 * 32 + 16)) + 4 * b.double().abs())
    assert float(((y - ref).abs() / bound).max()) <= 1


def test_log_probs_takes_whole_numbers():
    """(CPU: decided before the tensors are looked at.)  2.5 was taken for 2."""
    from erfnet_pytorch_amd import functional as hipf
    x, target = noise(4, 16), torch.zeros(4, dtype=torch.int64)
    for bad in (dict(top_k=2.5), dict(top_k=2.0), dict(top_k=2, ignore_index=0.5)):
        with pytest.raises(TypeError):
            hipf.log_probs(x, target, **bad)
    with pytest.raises(RuntimeError, match="cpu"):
        hipf.log_probs(x, target, top_k=torch.tensor(2), ignore_index=torch.tensor(-1))


# ================================================================================ sizes
@gpu
def test_log_probs_of_more_rows_than_a_launch_of_backward_holds():
    """2^24 + 12288 rows of 1025 bf16 classes (34 GB, and as much of a gradient): backward's blocks are more than HIP takes at once.
    The rows repeat every 4096, which begin at the same place of a cache line, so the results repeat bit for bit."""
    from erfnet_pytorch_amd import functional as hipf
    tile, times, v = 4096, 4099, 1025
    if torch.cuda.mem_get_info()[0] < 90 << 30:
        pytest.skip("needs 90 GB")
    piece, target = noise(tile, v, seed=5, dtype=torch.bfloat16).to(DEV), (torch.arange(tile) % v).to(DEV)
    g = noise(tile, seed=6).to(DEV)
    p = piece.clone().requires_grad_()
    few = hipf.log_probs(p, target, top_k=2)
    dp, = torch.autograd.grad((few.log_prob, few.entropy), p, (g, g))
    x = piece.repeat(times, 1).requires_grad_()
    r = hipf.log_probs(x, target.repeat(times), top_k=2)
    for a, b in zip(r, few):
        assert bool((a.detach().view(times, *b.shape) == b.detach()).all())
    dx, = torch.autograd.grad((r.log_prob, r.entropy), x, (g.repeat(times), g.repeat(times)))
    for part in dx.view(times, tile, v).split(256):
        assert bool((part == dp).all())


# ================================================================================ AdamW
@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_refuses_parameters_that_come_to_share_memory_later(bits):
    """Host parameters that come to the GPU on top of each other and have their state from a state dict; parameters that have
    stepped apart and are moved together.  Nothing is updated, counts included."""
    from erfnet_pytorch_amd import optim

    def pair(device):
        return [torch.nn.Parameter(torch.zeros(6, device=device)) for _ in range(2)]

    donor = pair(DEV)
    first = optim.AdamW(donor, state_bits=bits)
    for p in donor:
        p.grad = torch.ones_like(p)
    first.step()
    buf = torch.zeros(9, device=DEV)
    late = pair("cpu")
    opt = optim.AdamW(late, state_bits=bits)
    late[0].data, late[1].data = buf[:6], buf[3:]
    opt.load_state_dict(first.state_dict())
    for p in late:
        p.grad = torch.ones(6, device=DEV)
    with pytest.raises(ValueError, match="share memory"):
        opt.step()
    assert not buf.any() and all(float(opt.state[p]["step"]) == 1 for p in late)
    donor[1].data = donor[0].data
    with pytest.raises(ValueError, match="share memory"):
        first.step()
    donor[1].data = torch.zeros(6, device=DEV)
    first.step()
    assert all(float(first.state[p]["step"]) == 2 for p in donor)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_load_state_dict_minds_the_callers_hooks(bits):
    """(CPU.)  A hook before hands on another dict: that one is loaded.  A hook after sees the state as it stays, with the moments'
    own types, and what it does to it stays."""
    from erfnet_pytorch_amd import optim
    p = torch.nn.Parameter(noise(300, dtype=torch.bfloat16))
    opt = optim.AdamW([p], state_bits=bits)
    state = opt._new_state(p)
    key = opt._moments[0]
    saved = opt.state_dict()
    saved["state"] = {0: {**state, "step": torch.tensor(3.0)}}

    def before(optimizer, given):
        entry = given["state"][0]
        return {**given, "state": {0: {**entry, "step": entry["step"] + 4, key: torch.ones_like(entry[key], dtype=torch.float32).to(
            entry[key].dtype)}}}

    seen = []

    def after(optimizer):
        entry = optimizer.state[p]
        seen.append({k: v.dtype for k, v in entry.items()})
        entry["step"] += 10

    opt.register_load_state_dict_pre_hook(before)
    opt.register_load_state_dict_post_hook(after)
    for turn in (1, 2):
        opt.load_state_dict(saved)
        assert len(seen) == turn and seen[-1] == {k: v.dtype for k, v in state.items()}
        assert float(opt.state[p]["step"]) == 17 and bool((opt.state[p][key].float() == 1).all())
        assert opt.state[p][key].data_ptr() != saved["state"][0][key].data_ptr()
    bad = {**saved, "state": {0: {"step": torch.tensor(1.0)}}}
    with pytest.raises((ValueError, KeyError)):
        opt.load_state_dict(bad)
    opt.load_state_dict(saved)
    assert len(seen) == 3


def test_adamw_groups_are_refused_as_torch_refuses_them_and_hold_its_keys():
    """(CPU.)  A set has no order to put the state in; state_bits is the optimiser's, and was ignored where a group gave another."""
    import copy
    import pickle
    from erfnet_pytorch_amd import optim
    a, b, c = (torch.nn.Parameter(torch.zeros(3)) for _ in range(3))
    opt = optim.AdamW([a], state_bits=8)
    with pytest.raises(TypeError, match="ordered"):
        opt.add_param_group({"params": {b}})
    with pytest.raises(TypeError, match="dict"):
        opt.add_param_group([b])
    with pytest.raises(ValueError, match="state_bits"):
        opt.add_param_group({"params": [b], "state_bits": 32})
    with pytest.raises(ValueError, match="state_bits"):
        optim.AdamW([{"params": [a], "state_bits": 8}])
    assert len(opt.param_groups) == 1
    opt.add_param_group({"params": (p for p in [b]), "state_bits": 8, "lr": 1e-5})
    opt.add_param_group({"params": c})
    keys = set(torch.optim.AdamW([torch.nn.Parameter(torch.zeros(3))]).param_groups[0])
    for o in (opt, copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        assert o.state_bits == 8 and all(set(g) == keys for g in o.param_groups)
    assert [g["lr"] for g in opt.param_groups] == [1e-3, 1e-5, 1e-3]


@gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("eps", [2.0 ** -126, 1e-40, 2.0 ** -149, 1e-300])
def test_adamw_with_an_eps_below_the_normal_numbers(eps, bits):
    """No gradient so far: 0 / (0 + eps) = 0, however small eps is."""
    from erfnet_pytorch_amd import optim
    p = torch.nn.Parameter(noise(300).to(DEV))
    was = p.detach().clone()
    p.grad = torch.zeros_like(p)
    p.grad[::2] = 1.0
    optim.AdamW([p], lr=1e-2, eps=eps, weight_decay=0.0, state_bits=bits).step()
    assert torch.equal(p[1::2], was[1::2])
    # lr m / c1 / sqrt(v / c2) = lr: root, reciprocal and scalars to a few units each, and the difference's own rounding
    assert float((was[::2] - p.detach()[::2] - 1e-2).abs().max()) <= 32 * 2.0 ** -24 * 1e-2 + 2.0 ** -24 * 4


# ================================================================================ views that stand for their negative
def negative(t):
    """A contiguous view that stands for t, of memory that holds -t: what autograd leaves as the gradient of a single number that
    became the imaginary part of a complex one."""
    view = torch._neg_view(-t)
    assert view.is_neg() and view.is_contiguous()
    return view


@gpu
def test_gradient_of_a_number_in_complex_arithmetic_has_its_sign():
    from erfnet_pytorch_amd import optim
    p = torch.nn.Parameter(torch.zeros(1, device=DEV))
    z = torch.complex(torch.zeros(1, device=DEV), p)
    z.conj().backward(torch.full((1,), 1 + 2j, device=DEV))
    assert p.grad.is_neg() and float(p.grad) == -2
    optim.AdamW([p], lr=0.25, weight_decay=0.0).step()
    assert abs(float(p.detach()) - 0.25) < 1e-6


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_with_negated_views(bits):
    from erfnet_pytorch_amd import optim
    init, grad, new = noise(700, seed=1), noise(700, seed=2), []
    for wrap in (torch.clone, negative):
        p = torch.nn.Parameter(init.to(DEV))
        opt = optim.AdamW([p], state_bits=bits)
        for _ in range(2):
            p.grad = wrap(grad.to(DEV))
            opt.step()
        new.append(p.detach())
    assert torch.equal(*new)
    q = torch.nn.Parameter(negative(init.to(DEV)))
    q.grad = grad.to(DEV)
    if q.is_neg():
        with pytest.raises(ValueError, match="negative"):
            optim.AdamW([q], state_bits=bits).step()


@gpu
def test_layer_norm_and_log_probs_of_negated_views():
    from erfnet_pytorch_amd import functional as hipf
    t = {n: noise(*s, seed=i).to(DEV) for i, (n, s) in enumerate(
        dict(x=(4, 16), w=(16,), b=(16,), gy=(4, 16), image=(2, 8, 3, 5), logits=(4, 40), pixels=(2, 8, 3, 5), g=(4,), gp=(2, 3, 5)).items())}
    rows, map_ = torch.arange(4, device=DEV), torch.ones(2, 3, 5, dtype=torch.int64, device=DEV)

    def work(wrap):
        v = {n: wrap(a).requires_grad_() for n, a in t.items()}
        y = hipf.layer_norm(v["x"], v["w"], v["b"])
        out = [y, *torch.autograd.grad(y, (v["x"], v["w"], v["b"]), v["gy"].detach()), hipf.layer_norm(v["image"], dim=1)]
        for x, target, dim, g in ((v["logits"], rows, -1, v["g"]), (v["pixels"], map_, 1, v["gp"])):
            r = hipf.log_probs(x, target, top_k=2, dim=dim)
            out += [*r, *torch.autograd.grad((r.log_prob, r.entropy), x, (g.detach(), g.detach()))]
        return out

    for a, b in zip(work(torch.clone), work(negative)):
        assert torch.equal(a, b)


# ================================================================================ threads
@gpu
@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("op,entry", [("layer_norm", "erf_layer_norm_forward"), ("log_probs", "erf_log_probs_forward")])
def test_other_python_threads_run_while_a_call_waits(tmp_path, op, entry, grad):
    """The entry point is exchanged for one that sleeps, as a launch does whose queue is full."""
    import ctypes
    import subprocess
    import threading
    import time
    from erfnet_pytorch_amd import _lib, functional as hipf
    (tmp_path / "nap.c").write_text("#include <unistd.h>\nint nap(void) { usleep(500000); return 0; }\n")
    subprocess.run(["gcc", "-shared", "-fPIC", "nap.c", "-o", "nap.so"], cwd=tmp_path, check=True, timeout=60)
    nap = ctypes.CDLL(str(tmp_path / "nap.so")).nap
    x, target = noise(4, 16).to(DEV).requires_grad_(grad), torch.zeros(4, dtype=torch.int64, device=DEV)
    host, lib = _lib.host(), _lib.lib()

    def bind(other):
        host.bind(lambda name: ctypes.cast(other.get(name) or getattr(lib, name), ctypes.c_void_p).value)

    turns, done = [], threading.Event()

    def other():
        while not done.is_set():
            turns.append(time.monotonic())
            time.sleep(0.002)

    thread = threading.Thread(target=other)
    bind({entry: nap})
    try:
        thread.start()
        begin = time.monotonic()
        hipf.layer_norm(x) if op == "layer_norm" else hipf.log_probs(x, target)
        end = time.monotonic()
    finally:
        bind({})
        done.set()
        thread.join()
    assert end - begin > 0.4
    assert sum(begin + 0.05 < t < end - 0.05 for t in turns) > 20
    y = hipf.layer_norm(x.detach())
    assert float(y.mean(1).abs().max()) < 1e-6


@gpu
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,v", [(1301, 20011), (40_001, 701)])
def test_every_entry_of_a_streamed_gradient_equals_that_of_small_calls(rows, v, kind):
    """Gradients of 48 MB and more are stored past the caches, those of 576 rows are not.  576 rows begin at the same place of a
    cache line in both, and a row has the same threads at either count, so every entry is the same bit for bit."""
    from erfnet_pytorch_amd import functional as hipf
    g = torch.Generator(device=DEV).manual_seed(v)
    x = torch.randn(rows, v, generator=g, device=DEV).to(kind)
    t = torch.randint(0, v, (rows,), generator=g, device=DEV)
    ups = [torch.randn(rows, generator=g, device=DEV), torch.randn(rows, generator=g, device=DEV),
           torch.randn(rows, 3, generator=g, device=DEV)]
    assert x.nbytes >= 48 << 20 > 576 * v * x.element_size()

    def gradient(a, b):
        part = x[a:b].clone().requires_grad_()
        r = hipf.log_probs(part, t[a:b], 3)
        return torch.autograd.grad([r.log_prob, r.entropy, r.top_log_probs], part, [u[a:b] for u in ups])[0]

    whole = gradient(0, rows)
    for a in range(0, rows, 576):
        assert torch.equal(whole[a:a + 576], gradient(a, min(a + 576, rows))), a


@gpu
def test_every_entry_of_gradients_beyond_32_bit_offsets():
    """The last 288 of 32800 rows of 65537 classes (2^31 elements end within them) beside the same rows by themselves: as many
    blocks a row and the same place of a cache line, so all of dx is the same bit for bit, the small entries too."""
    from erfnet_pytorch_amd import functional as hipf
    v, rows, tail = 65537, 32800, 288
    g = torch.Generator(device=DEV).manual_seed(1)
    part = (3 * torch.randn(tail, v, generator=g, device=DEV)).bfloat16()
    t = torch.randint(0, v, (tail,), generator=g, device=DEV)
    ups = [torch.randn(tail, generator=g, device=DEV), torch.randn(tail, generator=g, device=DEV),
           torch.randn(tail, 4, generator=g, device=DEV)]
    x = torch.zeros(rows, v, dtype=torch.bfloat16, device=DEV)
    x[-tail:] = part
    assert (rows - tail) * v < 1 << 31 < rows * v and (rows - tail) * v * 2 % 128 == 0

    def run(x, t, ups):
        x = x.requires_grad_()
        r = hipf.log_probs(x, t, 4)
        return [*(o.detach()[-tail:] for o in r),
                torch.autograd.grad([r.log_prob, r.entropy, r.top_log_probs], x, ups)[0][-tail:]]

    def padded(u):
        return torch.cat([u.new_zeros(rows - tail, *u.shape[1:]), u])

    for a, b in zip(run(x, padded(t), [padded(u) for u in ups]), run(part, t, ups)):
        assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("c", [20, 1000, 5000])
def test_layer_norm_with_a_variance_below_the_normal_numbers(c, kind):
    """Equal values and an eps of 1e-40: y = bias, dx = (g - mean g) / sqrt(eps) (eps rounds to 2^-149 in fp32: 1e-5 of itself).
    Spreads of 2^-66 and no eps: the squares keep 2^-18 of themselves (they are near 2^-132, rounded to 2^-149), the
    root half of that; the rest is as ever."""
    from erfnet_pytorch_amd import functional as hipf
    own, u = (0.0 if kind == torch.float32 else 2.0 ** -8), 2.0 ** -24
    b = noise(c, seed=1)
    g = noise(3, c, seed=2, dtype=kind)
    x = torch.full((3, c), 0.75, dtype=kind).to(DEV).requires_grad_()
    y = hipf.layer_norm(x, None, b.to(DEV), eps=1e-40)
    assert torch.equal(y, b.to(DEV).to(kind).expand_as(y))
    dx, = torch.autograd.grad(y, x, g.to(DEV))
    mean = g.double().mean(1, keepdim=True)
    ref, size = (g.double() - mean) * 1e20, (g.double().abs() + g.double().abs().mean(1, keepdim=True)) * 1e20
    assert float(((dx.cpu().double() - ref).abs() - (2e-5 + 72 * u) * size * (1 + own) - own * ref.abs()).max()) <= 0
    x = noise(3, c, seed=c, dtype=kind) * 2.0 ** -66
    y = hipf.layer_norm(x.to(DEV), eps=0.0).cpu().double()
    d = x.double() - x.double().mean(1, keepdim=True)
    ref = d / torch.sqrt((d * d).mean(1, keepdim=True))
    assert float(((y - ref).abs() - (2.0 ** -18 + 72 * u) * (1 + ref.abs()) * (1 + own) - own * ref.abs()).max()) <= 0


@gpu
def test_two_threads_call_at_once_on_streams_of_their_own():
    import threading
    from erfnet_pytorch_amd import functional as hipf, optim
    target = torch.arange(9, device=DEV)

    def work(seed):
        x, w = noise(9, 3000, seed=seed).to(DEV), torch.nn.Parameter(1 + 0.1 * noise(3000, seed=seed + 1).to(DEV))
        opt = optim.AdamW([w], lr=1e-2, state_bits=8 if seed % 2 else 32)
        for _ in range(20):
            w.grad = None
            r = hipf.log_probs(hipf.layer_norm(x, w), target, 4)
            (r.log_prob.sum() + r.entropy.sum() + r.top_log_probs.sum()).backward()
            opt.step()
        return w.detach()

    alone = [work(s) for s in (1, 2)]
    got = [None, None]

    def thread(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            got[i] = work(i + 1)
        stream.synchronize()

    threads = [threading.Thread(target=thread, args=(i,)) for i in range(2)]
    torch.cuda.synchronize()
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(alone, got):
        assert torch.equal(a, b)
