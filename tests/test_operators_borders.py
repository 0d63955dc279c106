"""The learner-step operators where they could go wrong without the tests of test_operators.py showing it: precision against the f32 form's, values at the
types' borders, ways of calling that autograd, tracing and views allow, and rows enough for every loop."""
import math

import pytest
import torch

from test_operators import U, half_step


# ------------------------------------------------------------------------------------------------------------ orthogonalize

def iteration(g, dtype, steps=5, eps=1e-7):
    """The Newton-Schulz iteration in elementary products of one type, on the side with fewer rows."""
    tall = g.shape[0] > g.shape[1]
    x = (g.T if tall else g).to(dtype)
    x = x / (x.double().square().sum().sqrt() + eps).to(dtype)
    for _ in range(steps):
        a = x @ x.T
        x = 3.4445 * x + (-4.7750 * a + 2.0315 * (a @ a)) @ x
    return x.T if tall else x


def gradient_like(m, n, kind, seed):
    """randn: all singular values alike; decay: falling like a Linear's gradient; rank8: eight directions and 1 % noise; steep: down to a thousandth."""
    gen = torch.Generator('cuda').manual_seed(seed)
    normal = lambda *s: torch.randn(s, generator=gen, device='cuda', dtype=torch.float64)
    q = min(m, n)
    if kind == 'randn':
        return normal(m, n)
    if kind == 'decay':
        return .01 * (normal(m, q) * torch.arange(1, q + 1, device='cuda').double().rsqrt()) @ normal(q, n) / q
    if kind == 'rank8':
        return normal(m, 8) @ normal(8, n) + .01 * normal(m, n)
    u, v = torch.linalg.qr(normal(m, q))[0], torch.linalg.qr(normal(n, q))[0]
    return (u * torch.logspace(-3, 0, q, device='cuda', dtype=torch.float64)) @ v.T


KINDS = ['randn', 'decay', 'rank8', 'steep']
FEW = [(1, 1), (1, 700), (2, 500), (8, 8), (8, 129), (129, 8), (8, 4000), (16, 16), (16, 162), (17, 256), (17, 257), (32, 200), (200, 32), (33, 300), (48, 129), (64, 200), (63, 1001),
       (1001, 63), (3, 16384), (5000, 40)]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize('m,n', FEW)
def test_few_rows_are_exact_but_for_the_last_rounding(m, n, dtype):
    """Up to 32 rows (columns), or 64 beside more than 128, are computed in f64: an entry is off by its rounding, through f32, and by what f64 leaves.  A Gram matrix is a random
    walk of n + 20 m roundings off; the steps' product takes a deviation of A to at most 5e4 times that of the result (the derivative of the five steps'
    polynomial, 1.5e7 at 0 and falling, times the square root of the eigenvalue); four deviations of the walk."""
    from boardlaw_amd import optim
    mats = [gradient_like(m, n, kind, m + n).to(dtype) for kind in KINDS]
    for kind, g, o in zip(KINDS, mats, optim.orthogonalize(mats)):
        want = iteration(g, torch.float64)
        tol = (half_step(dtype) + U) * want.abs() + 5e4 * 4 * (n + m + 20 * min(m, n)) ** .5 * 2. ** -53 + torch.finfo(dtype).tiny * half_step(dtype) * 2
        off = (o.double() - want).abs() / tol
        assert o.dtype == dtype and off.max() <= 1, (kind, float(off.max()))


@pytest.mark.gpu
@pytest.mark.parametrize('count,m,n', [(3, 20, 24), (3, 20, 700), (40, 600, 20), (3, 64, 1000), (3, 50, 60), (3, 100, 150), (35, 130, 140)])
def test_orthogonalize_in_place(count, m, n):
    """The C entry point may write over its input; more matrices than one launch takes, each its own."""
    import ctypes
    from boardlaw_amd import _native, optim
    L = _native.lib()
    mats = [gradient_like(m, n, KINDS[i % 4], i).float() for i in range(count)]
    want = [optim.orthogonalize(g) for g in mats]
    assert all(torch.equal(a, b) for a, b in zip(optim.orthogonalize(mats), want))
    work = torch.empty(L.bl_orthogonalize_workspace(count, m, n), dtype=torch.uint8, device='cuda')
    at = (ctypes.c_void_p * count)(*[g.data_ptr() for g in mats])
    _native.check(L.bl_orthogonalize(at, at, count, 0, m, n, 5, 1e-7, work.data_ptr(), torch.cuda.current_stream().cuda_stream))
    assert all(torch.equal(a, b) for a, b in zip(mats, want))


@pytest.mark.gpu
@pytest.mark.parametrize('m,n', [(1, 1), (20, 24), (700, 20), (50, 60), (50, 100), (100, 150), (512, 512)])
def test_orthogonalize_of_nothing(m, n):
    """A zero matrix gives zeros with any eps, none among them, beside others; NaN and infinities take their own matrix only."""
    from boardlaw_amd import optim
    one = gradient_like(m, n, 'randn', 1).float()
    nan, inf = one.clone(), one.clone()
    nan[m // 2, n // 2], inf[-1, -1] = math.nan, math.inf
    for eps in (0., 1e-7, 1e-45):
        for dtype in (torch.float32, torch.float16, torch.bfloat16):
            z, a, b, c = optim.orthogonalize([t.to(dtype) for t in (torch.zeros_like(one), one, nan, inf)], eps=eps)
            assert (z == 0).all() and b.isnan().all() and c.isnan().all()
            want = iteration(one.to(dtype), torch.float64, eps=eps)
            assert (a.double() - want).norm() <= (half_step(dtype) + 2e-5) * want.norm()        # (the value itself: tested elsewhere)


# ------------------------------------------------------------------------------------------------- ways of calling

def calls(device):
    """Each operator as a function of one tensor."""
    from boardlaw_amd import heads, networks, optim
    w = torch.ones(4, device=device)
    base = torch.ones((3, 4), device=device)
    return dict(logprobs=lambda t: heads.logprobs(t, k=2).entropy, stream=lambda t: networks.norm_residual(t, base, None, w, pre=w)[1],
                branch=lambda t: networks.norm_residual(base, t, None, w, pre=w)[0], gate=lambda t: networks.norm_residual(base, base, gate=t)[0],
                norm=lambda t: networks.norm_residual(t, pre=w)[1], orthogonalize=lambda t: optim.orthogonalize([t])[0])


@pytest.mark.parametrize('name', ['logprobs', 'stream', 'branch', 'gate', 'norm', 'orthogonalize'])
@pytest.mark.parametrize('device', ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)])
def test_what_would_be_lost_is_refused(name, device):
    """A tangent (also of a tensor that requires no gradient) and a tracer's call raise: the operators know neither.  Refused before the device is looked at."""
    from torch.autograd import forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx
    f = calls(device)[name]
    x = torch.randn((3, 4), device=device)
    with forward_ad.dual_level():
        for leaf in (x, x.clone().requires_grad_()):
            dual = forward_ad.make_dual(leaf, torch.ones_like(x))
            with pytest.raises(NotImplementedError, match='tangent'):
                f(dual)
            with torch.no_grad(), pytest.raises(NotImplementedError, match='tangent'):
                f(dual)
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.jvp(f, (x,), (x,))
    with pytest.raises(RuntimeError):
        torch.func.vmap(f)(x[None].expand(2, 3, 4))
    with pytest.raises(NotImplementedError, match='traced'):
        torch.jit.trace(f, (x,), check_trace=False)
    with pytest.raises(NotImplementedError, match='traced'):
        make_fx(f)(x)


@pytest.mark.gpu
@pytest.mark.parametrize('name', ['logprobs', 'stream', 'branch', 'gate', 'norm'])
def test_a_backward_pass_is_not_traced(name):
    from torch.fx.experimental.proxy_tensor import make_fx
    x = torch.randn((3, 4), device='cuda', requires_grad=True)
    out = calls('cuda')[name](x)
    with pytest.raises(NotImplementedError, match='traced'):
        make_fx(lambda g: torch.autograd.grad(out, x, g, retain_graph=True))(torch.ones_like(out))
    torch.autograd.grad(out, x, torch.ones_like(out))


@pytest.mark.gpu
def test_tensors_whose_sign_is_a_flag():
    """The imaginary part of a conjugated tensor, dense or not, as any input and as a gradient: its values count, not what lies in memory."""
    from boardlaw_amd import heads, networks, optim

    def flagged(*shape):
        z = torch.complex(torch.randn(shape, device='cuda'), torch.randn(shape, device='cuda'))
        t = z.conj().imag
        assert t.is_neg()
        return t

    dense = lambda t: torch._neg_view(t)
    for W in (1, 12):
        for lazy in (flagged(5, W), dense(torch.randn((5, W), device='cuda'))):
            real = lazy.clone()
            assert lazy.is_neg() and not real.is_neg()
            same = lambda f: all(torch.equal(a, b) for a, b in zip(f(lazy), f(real)))
            assert same(lambda t: heads.logprobs(t, torch.zeros(5, dtype=torch.int64, device='cuda'), k=2).values())
            base, one = torch.randn((5, W), device='cuda'), torch.ones(W, device='cuda')
            assert same(lambda t: networks.norm_residual(t, base, pre=one)) and same(lambda t: networks.norm_residual(base, t, pre=one))
            assert same(lambda t: networks.norm_residual(base, base, gate=t)[:1]) and same(lambda t: networks.norm_residual(base, base, gate=t[:, :1])[:1])
            assert same(lambda t: networks.norm_residual(base, base, None, t[0], t[1], t[2])) and same(lambda t: networks.norm_residual(base, base, t[0, 0])[:1])
            assert same(lambda t: [optim.orthogonalize(t)])

            def gradients(t):
                x = base.detach().requires_grad_()
                out, h = networks.norm_residual(x, base, pre=one)
                o = heads.logprobs(x)
                return torch.autograd.grad([out, h], x, [t, t], retain_graph=True) + torch.autograd.grad(o.entropy, x, t[:, 0])

            assert same(gradients)
    a = dense(torch.tensor([0, -3], device='cuda'))
    x = torch.randn((2, 5), device='cuda')
    assert torch.equal(heads.logprobs(x, a).logp, heads.logprobs(x, torch.tensor([0, 3], device='cuda')).logp)


# ------------------------------------------------------------------------------------------------- a learner's step

@pytest.mark.parametrize('where', ['policy.core.weight', 'body.1.weight'])
@pytest.mark.parametrize('device,kind', [('cpu', 'list'), ('cpu', 'several'), pytest.param('cuda', 'muon', marks=pytest.mark.gpu)])
def test_an_overflow_skips_every_optimiser(where, device, kind):
    """An infinite gradient in one optimiser's parameters: no parameter moves and the scale goes down, as with one optimiser; then a step of all."""
    from boardlaw_amd import arrdict, heads, networks, optim, training, validation
    torch.manual_seed(0)
    net = networks.FCModel(heads.Tensor((1,)), heads.Masked(2), width=8, depth=2).to(device)
    with torch.no_grad():
        for p in net.parameters():
            if p.ndim == 0:
                p.fill_(.4)
    worlds = validation.All.initial(n_envs=16, n_seats=1, length=4, device=device)
    logits = torch.log_softmax(torch.randn((16, 2), device=device), -1)
    batch = arrdict.arrdict(worlds=worlds, decisions=arrdict.arrdict(logits=logits.half(), v=torch.randn((16, 1), device=device).half()), reward_to_go=torch.randn((16, 1), device=device).half())
    hidden, rest = optim.split(net)
    opt = training.make_optimizer(net, 'muon') if kind == 'muon' else [torch.optim.SGD(hidden, lr=.1), torch.optim.Adam(rest, lr=.1)]
    opt = optim.Several(opt) if kind == 'several' else opt
    scaler = torch.amp.GradScaler(device, init_scale=4., growth_interval=100)
    before = {k: v.clone() for k, v in net.state_dict().items()}
    hook = dict(net.named_parameters())[where].register_hook(lambda g: g * math.inf)
    training.optimize(net, scaler, opt, batch)
    assert all(torch.equal(v, before[k]) for k, v in net.state_dict().items()) and scaler.get_scale() == 2.
    assert not any(o.state for o in opt)
    hook.remove()
    training.optimize(net, scaler, opt, batch)
    after = net.state_dict()
    assert not torch.equal(after['policy.core.weight'], before['policy.core.weight']) and not torch.equal(after['body.1.weight'], before['body.1.weight'])
    assert all(torch.isfinite(v).all() for v in after.values()) and scaler.get_scale() == 2.
