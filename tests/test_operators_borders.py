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


# ------------------------------------------------------------------------------------------------------------ norm_residual

@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize('W', [2, 20, 100, 512, 600, 771, 1024, 1500, 4096, 8191, 8192])
def test_norms_of_the_largest_and_smallest_rows(W, dtype):
    """Rows whose sum of squares leaves f32's range, beside ordinary ones: h is pre times something of size 1 all the same, and every gradient the
    formula's.  Seven rows: one of a shared wave or workgroup is extreme where the others are not."""
    from boardlaw_amd import networks
    torch.manual_seed(W)
    base = torch.randn((7, W), device='cuda')
    pre, post = 1 + .2 * torch.randn(W, device='cuda'), 1 + .2 * torch.randn(W, device='cuda')
    gx = torch.randn((7, W), device='cuda')
    # a row's sums: up to 24 + W / 512 roundings, as for ordinary rows; the scales are powers of two
    k = 40 + W / 256
    for powers, eps in (((0, 64, 100, 1, 70, 0, 122), 1e-5), ((0, -60, -100, 1, -80, 0, -118), 0.)):
        scale = torch.tensor([2. ** p for p in powers], device='cuda', dtype=torch.float64)[:, None]
        x = (base.double() * scale).to(dtype)
        # the norm before a block
        leaf = x.detach().requires_grad_()
        _, h = networks.norm_residual(leaf, pre=pre, eps=eps)
        g = gx.to(dtype)
        d, = torch.autograd.grad(h, leaf, g)
        want = x.double().requires_grad_()
        rms = (want.square().mean(-1, keepdim=True) + eps).sqrt()
        wh = pre.double() * want / rms
        wd, = torch.autograd.grad(wh, want, g.double(), retain_graph=True)
        assert (h.double() - wh).abs().le((half_step(dtype) + U * k) * wh.abs()).all()
        # (the gradient's terms are of size |g pre| / rms, and cancel; beyond 2^100 it is a subnormal number or none: half of f32's smallest step)
        size = (g.double() * pre).abs() / rms + (wh / pre).abs() * ((g.double() * wh).abs().mean(-1, keepdim=True) / rms)
        assert (d.double() - wd).abs().le(half_step(dtype) * wd.abs() + U * 2 * k * size + 2. ** -133).all()
        # the norm behind it: n is of size 1
        leaf = x.detach().requires_grad_()
        stream = torch.zeros((7, W), device='cuda', dtype=dtype)
        out, _ = networks.norm_residual(stream, leaf, None, post, eps=eps)
        d, = torch.autograd.grad(out, leaf, g)
        wn = post.double() * want / rms
        wd, = torch.autograd.grad(wn, want, g.double())
        assert (out.double() - wn).abs().le((half_step(dtype) + U * k) * wn.abs()).all()
        size = (g.double() * post).abs() / rms + (wn / post).abs() * ((g.double() * wn).abs().mean(-1, keepdim=True) / rms)
        assert (d.double() - wd).abs().le(half_step(dtype) * wd.abs() + U * 2 * k * size + 2. ** -133).all()
    # the extreme rows do not touch the others
    x = base.clone()
    plain = networks.norm_residual(x, pre=pre)[1]
    x[3] *= 2. ** 100
    other = networks.norm_residual(x, pre=pre)[1]
    keep = [0, 1, 2, 4, 5, 6]
    assert torch.equal(plain[keep], other[keep])


@pytest.mark.gpu
@pytest.mark.parametrize('tx,ty', [(torch.float32, torch.float32), (torch.float32, torch.float16), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16)], ids=str)
@pytest.mark.parametrize('W', [24, 90, 512, 700, 2000, 8192])
def test_blocks_with_extreme_rows(W, tx, ty):
    """The whole operator with every kind of gate on a stream, and a branch, of which some rows leave the range of squares."""
    from boardlaw_amd import networks
    from test_operators import norm_inputs, plain_norm
    R = 9
    k = 60 + W / 256
    for kind in ('none', 'packed', 'full', 'channel', 'row'):
        t, _ = norm_inputs(R, W, tx, ty, kind)
        t['x'][4] = (t['x'][4].double() * 2. ** 90).to(tx)
        if ty != torch.float16:
            t['y'][7, :W] = (t['y'][7, :W].double() * 2. ** 90).to(ty)
        with torch.no_grad():
            for drop in ((), ('post',), ('pre',), ('alpha',)):
                s = {n: None if n in drop else v for n, v in t.items()}
                if 'post' in drop and ty != torch.float16:
                    s['alpha'] = t['alpha'] * 2. ** -20                     # (the branch as it is)
                out, h = networks.norm_residual(**s)
                wo, wh = plain_norm(s['x'], s['y'], s['alpha'], s['post'], s['gate'], s['pre'], 1e-5)
                size = wo.abs() + (wo - s['x'].double()).abs()
                assert (out.double() - wo).abs().le(half_step(tx) * wo.abs() + U * k * size).all(), (kind, drop)
                if wh is not None:
                    # x_out's cancellation, through 1 / rms
                    scale = wh.abs() + size * (s['pre'].double().abs() / (wo.square().mean(-1, keepdim=True) + 1e-5).sqrt())
                    assert (h.double() - wh).abs().le(half_step(ty) * wh.abs() + 2 * U * k * scale + torch.finfo(ty).tiny * half_step(ty) * 2).all(), (kind, drop)


@pytest.mark.gpu
@pytest.mark.parametrize('hook', ['on the cpu', 'transposed', 'checkpoint'])
def test_saved_tensors_may_come_back_from_hooks(hook):
    """What is saved for the backward pass goes through saved-tensor hooks, which may return it elsewhere in memory and with other strides: the same gradients.
    (But for the order of sums: the columns from 5 on lie on 16-byte boundaries when they come back.  An entry's sums over 40 columns and 40 rows then differ
    by 64 roundings each way of terms as large as the tensor's largest entry, a few of them joined, and can round to f16's next value.)"""
    from torch.utils.checkpoint import checkpoint
    from boardlaw_amd import heads, networks
    torch.manual_seed(0)
    wide, both = torch.randn((40, 3 * 48), device='cuda'), torch.randn((40, 2 * 40), device='cuda').half()
    valid, actions = torch.rand((1, 48), device='cuda') < .8, torch.randint(0, 48, (40,), device='cuda')
    alpha, post, pre, channel = torch.tensor(.7, device='cuda'), torch.rand(40, device='cuda'), torch.rand(40, device='cuda'), torch.randn(40, device='cuda')
    element = torch.randn((40, 40), device='cuda').half()

    def f(a, x, y, al, po, pr, ch, el):
        o = heads.logprobs(a[:, 48:96], actions, valid, k=3)
        return (o.logp, o.entropy, o.top_logp, *networks.norm_residual(x[:, 5:45], y, al, po, pre=pr), *networks.norm_residual(x[:, :40], y[:, :40], al, po, ch, pr),
                *networks.norm_residual(x[:, :40], y[:, :40], al, po, el, pr))

    def gradients(run, context):
        leaves = [t.detach().clone().requires_grad_() for t in (wide, wide, both, alpha, post, pre, channel, element)]
        torch.manual_seed(1)
        with context:
            outs = run(*leaves)
        return torch.autograd.grad(outs, leaves, [torch.randn(o.shape, device='cuda').to(o.dtype) for o in outs])

    import contextlib
    turned = lambda t: t.t().contiguous().t() if t.dim() == 2 else torch.stack([t, t], -1)[..., 0]
    context = {'on the cpu': lambda: torch.autograd.graph.save_on_cpu(), 'checkpoint': contextlib.nullcontext,
               'transposed': lambda: torch.autograd.graph.saved_tensors_hooks(turned, lambda t: t)}[hook]()
    run = f if hook != 'checkpoint' else lambda *leaves: checkpoint(f, *leaves, use_reentrant=False)
    want = gradients(f, contextlib.nullcontext())
    for a, b in zip(gradients(run, context), want):
        assert (a.float() - b.float()).abs().le(4 * 64 * U * b.float().abs().amax() + 2 * half_step(b.dtype) * b.float().abs()).all()


def formula(t, g_out, g_h, eps=1e-5):
    """networks.norm_residual and its gradients in 64 bits from their formulas, each with the sum of its terms' sizes (a term's own error is of its size: x_out's
    cancellation counts with the sizes of what it is made of)."""
    W = t['x'].shape[-1]
    d = {n: None if v is None else v.detach().double() for n, v in t.items()}
    x, alpha, post, pre = d['x'], d['alpha'], d['post'], d['pre']
    y, gate = (d['y'][:, :W], d['y'][:, W:]) if d['y'].shape[-1] == 2 * W else (d['y'], d['gate'])
    mean = lambda v: v.mean(-1, keepdim=True)
    ry = 1 / (mean(y * y) + eps).sqrt()
    n, s = y * ry, 1. if gate is None else torch.sigmoid(gate).expand_as(y)
    u = s * post * n
    out = x + alpha * u
    rx = 1 / (mean(out * out) + eps).sqrt()
    xn, xs = out * rx, (x.abs() + (alpha * u).abs()) * rx
    gx, gh = g_out.double(), g_h.double()
    tt = gh * pre
    z, zs = gx + rx * (tt - xn * mean(tt * xn)), gx.abs() + rx * (tt.abs() + xs * mean((tt * xs).abs()))
    dn, dns = alpha * z * s * post, (alpha * s * post).abs() * zs
    dy, dys = ry * (dn - n * mean(dn * n)), ry * (dns + n.abs() * mean(dns * n.abs()))
    want = dict(x=(z, zs), alpha=((z * u).sum(), (zs * u.abs()).sum()), post=((alpha * z * s * n).sum(0), ((alpha * s * n).abs() * zs).sum(0)), pre=((gh * xn).sum(0), (gh.abs() * xs).sum(0)))
    if gate is not None:
        dg, dgs = alpha * z * post * n * s * (1 - s), (alpha * post * n).abs() * zs * s * (1 - s)
    if d['y'].shape[-1] == 2 * W:
        dy, dys = torch.cat([dy, dg], -1), torch.cat([dys, dgs], -1)
    elif gate is not None:
        want['gate'] = (dg, dgs) if gate.shape == y.shape else (dg.sum(0), dgs.sum(0)) if gate.ndim == 1 else (dg.sum(-1, keepdim=True), dgs.sum(-1, keepdim=True))
    want['y'] = dy, dys
    return (out, x.abs() + (alpha * u).abs()), (pre * xn, pre.abs() * xs), want


# more rows than one pass of all workgroups, forward (2048 workgroups) and backward (512), and a rest; 4, 16, 64, 128, 256, 512 and 1024 lanes a row
MANY_ROWS = [(131200, 20), (131137, 24), (32900, 81), (33001, 88), (8300, 300), (8259, 512), (4201, 771), (4101, 776), (2100, 1501), (2099, 2048), (2061, 3001), (2070, 4096), (2055, 8191), (2051, 8192)]


@pytest.mark.gpu
@pytest.mark.parametrize('R,W', MANY_ROWS)
def test_norm_residual_of_many_rows(R, W):
    """Every entry, and every column's sum over the rows, to within what its own terms allow: a row's sums have up to 24 + W / 512 roundings and every
    term a few of them joined; a sum over rows one more for each of a lane's rows (under 8), a workgroup's 64 groups of lanes, 32 workgroups of a part, and 16 parts."""
    from boardlaw_amd import networks
    from test_operators import norm_inputs
    k = 4 * (24 + W / 512)
    for (tx, ty), kind in ((torch.float32, torch.float32), 'channel'), ((torch.float32, torch.float16), 'packed'), ((torch.bfloat16, torch.bfloat16), 'full'), ((torch.float32, torch.bfloat16), 'row'):
        t, n = norm_inputs(R, W, tx, ty, kind)
        t['y'][:, W // 3] *= 2. ** -12                                       # a small column beside the others
        names = [a for a in t if t[a] is not None]
        leaves = [t[a].requires_grad_() for a in names]
        out, h = networks.norm_residual(**t)
        g_out, g_h = (n(R, W) + .25 * t['y'][:, :W].detach().float()).to(tx), n(R, W).to(ty)
        grads = dict(zip(names, torch.autograd.grad([out, h], leaves, [g_out, g_h])))
        with torch.no_grad():
            wo, wh, want = formula(t, g_out, g_h)
            for name, got, (w, size), rows in [('out', out, wo, 0), ('h', h, wh, 0)] + [(a, grads[a], want[a], 0 if grads[a].shape[0:1] == (R,) else 120) for a in names]:
                tol = half_step(got.dtype) * w.abs() + U * (k + rows) * size + torch.finfo(got.dtype).tiny * half_step(got.dtype) * 2
                off = float(((got.double() - w).abs() / tol).max())
                assert off <= 1, (kind, name, off)
        del out, h, grads, want, wo, wh


# ------------------------------------------------------------------------------------------------------- orthogonalize, larger

@pytest.mark.gpu
@pytest.mark.parametrize('count,m,n', [(1, 33, 40), (2, 48, 64), (1, 64, 64), (2, 64, 128), (2, 100, 50), (1, 65, 65), (2, 65, 1000), (1, 100, 700), (3, 162, 512), (2, 512, 162), (1, 257, 257),
                                       (35, 130, 140), (4, 512, 512), (9, 512, 512), (26, 512, 512), (3, 1280, 1280), (6, 1024, 512), (8, 1024, 1024)])
def test_orthogonalize_is_as_exact_as_f32_products(count, m, n):
    """Operands of 22 (33) bits and f32 sums: against 64 bits no more than 1.5 times as far off as the iteration in f32 products, on every spectrum; the low-rank
    ones with noise are where operands of fewer bits fail (pairs of bf16 numbers: 40 times).  A matrix of its own spectrum each, more than one launch takes."""
    from boardlaw_amd import optim
    mats = [gradient_like(m, n, KINDS[i % 4], i).float() for i in range(max(count, 4))]
    outs = optim.orthogonalize(mats[:count]) if count >= 4 else [optim.orthogonalize([g])[0] for g in mats]
    for i, (g, o) in enumerate(zip(mats, outs)):
        if i >= 12 and i % 8:
            continue
        want = iteration(g, torch.float64)
        own, plain = float((o.double() - want).norm() / want.norm()), float((iteration(g, torch.float32).double() - want).norm() / want.norm())
        assert own <= 1.5 * plain + U, (KINDS[i % 4], own / plain)


# ------------------------------------------------------------------------------------------------- capture and build

@pytest.mark.gpu
def test_moves_are_captured_while_another_thread_asks_its_events():
    """As an nccl process group's watchdog does: the captured moves are the eager ones, and the other thread sees no error."""
    import threading
    from boardlaw_amd import hex, networks
    from boardlaw_amd.mcts import MCTSAgent
    worlds = hex.Hex.initial(8, 4)
    torch.manual_seed(0)
    net = networks.FCModel(worlds.obs_space, worlds.action_space, width=16, depth=1).cuda()
    event, done, errors, asked = torch.cuda.Event(), threading.Event(), [], []
    event.record()
    torch.cuda.synchronize()

    def ask():
        while not done.is_set():
            try:
                asked.append(event.query())
            except Exception as e:
                errors.append(e)
                return

    thread = threading.Thread(target=ask)
    thread.start()
    try:
        agent = MCTSAgent(net, n_nodes=8, graph=True)
        agent(worlds)
        torch.manual_seed(3)
        got = agent(worlds)
        torch.cuda.synchronize()
    finally:
        done.set()
        thread.join(30)
    assert not errors and asked
    eager = MCTSAgent(net, n_nodes=8)
    eager(worlds)
    torch.manual_seed(3)
    want = eager(worlds)
    assert torch.equal(got.actions, want.actions) and torch.equal(got.logits, want.logits)


def test_no_packed_fp32_instructions(tmp_path):
    """The build's flags keep the compiler from making them of ordinary float code, where it would."""
    import subprocess
    from boardlaw_amd import build
    src = tmp_path / 'x.hip'
    src.write_text('#include <hip/hip_runtime.h>\n__global__ void k(float2* x, float2 a) { float2 v = x[threadIdx.x]; v.x = v.x * a.x + a.y; v.y = v.y * a.x + a.y; '
                   'x[threadIdx.x] = make_float2(v.x + a.x, v.y + a.x); }\n')
    listing = lambda flags: subprocess.run([build._hipcc(), *flags, '-w', '--cuda-device-only', '-S', str(src), '-o', '-'], check=True, capture_output=True, text=True).stdout
    flags = [f for f in build.FLAGS if f not in ('-Xclang', '-target-feature', '-packed-fp32-ops')]
    packed = ('v_pk_add_f32', 'v_pk_mul_f32', 'v_pk_fma_f32')
    assert any(p in listing(flags) for p in packed) and not any(p in listing(build.FLAGS) for p in packed)


@pytest.mark.gpu
@pytest.mark.parametrize('change', ['device', 'shape', 'type'])
def test_saved_tensors_that_came_back_changed_are_refused(change):
    """A hook that returns a saved tensor elsewhere, shorter or as another type: an error before anything is launched.  One tensor at a time."""
    from boardlaw_amd import heads, networks
    alter = dict(device=lambda t: t.cpu(), shape=lambda t: t[..., :-1] if t.dim() else t[None], type=lambda t: t.double() if t.is_floating_point() else t.int())[change]
    x, y, w = torch.randn((6, 8), device='cuda'), torch.randn((6, 8), device='cuda').half(), torch.rand(8, device='cuda')
    valid, actions = torch.ones((6, 8), dtype=torch.bool, device='cuda'), torch.zeros(6, dtype=torch.int64, device='cuda')
    calls = [lambda: heads.logprobs(x.requires_grad_(), actions, valid, k=2).entropy]
    calls += [lambda gate=gate: networks.norm_residual(x.requires_grad_(), y, torch.tensor(.5, device='cuda'), w, gate, w)[1] for gate in (y, w, y[:, :1], None)]
    calls += [lambda: networks.norm_residual(x.requires_grad_(), torch.cat([y, y], -1), pre=w)[0], lambda: networks.norm_residual(x.requires_grad_(), pre=w)[1],
              lambda: heads.logprobs(x.requires_grad_(), k=2).top_logp]
    for call in calls:
        count, at = 0, 0
        while at <= count:                                                   # the at-th saved tensor; once more with none
            seen = []
            with torch.autograd.graph.saved_tensors_hooks(lambda t: (len(seen), seen.append(0), t)[::2], lambda p: alter(p[1]) if p[0] == at else p[1]):
                out = call()
            count = len(seen)
            if at < count:
                with pytest.raises(RuntimeError, match='saved tensor|Expected all tensors'):
                    torch.autograd.grad(out.sum(), x)
            else:
                torch.autograd.grad(out.sum(), x)
            at += 1
        assert count >= 3


@pytest.mark.gpu
def test_compiled_and_inference_mode_calls():
    """torch.compile leaves the operators outside its graphs, and inference mode needs nothing of autograd: the eager results."""
    f = calls('cuda')
    for name, call in f.items():
        x = torch.randn((3, 4), device='cuda')
        want = call(x)
        with torch.inference_mode():
            assert torch.equal(call(x), want) and torch.equal(call(x.clone()), want)
        torch._dynamo.reset()
        assert torch.equal(torch.compile(lambda t: 2 * call(t + 0), backend='eager')(x), 2 * want)


@pytest.mark.gpu
@pytest.mark.parametrize('m,n', [(16, 16), (20, 700), (64, 300), (50, 60)])
def test_few_rows_on_streams_and_in_graphs(m, n):
    """Two captured graphs, replayed in turn on new matrices between eager calls on two streams: every result the eager one's."""
    from boardlaw_amd import optim
    mats = lambda seed: [gradient_like(m, n, KINDS[i % 4], 10 * seed + i).float() for i in range(5)]
    want = {s: optim.orthogonalize(mats(s)) for s in range(4)}
    graphs = []
    for _ in range(2):
        static = mats(0)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            optim.orthogonalize(static)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = optim.orthogonalize(static)
        graphs.append((graph, static, outs))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in (1, 2, 3, 1):
        inputs = mats(s)
        torch.cuda.synchronize()
        got = []
        for stream in streams:
            with torch.cuda.stream(stream):
                got.append(optim.orthogonalize(inputs))
        for graph, static, outs in graphs:
            for dst, src in zip(static, inputs):
                dst.copy_(src)
            graph.replay()
        torch.cuda.synchronize()
        for result in got + [outs for _, _, outs in graphs]:
            assert all(torch.equal(a, b) for a, b in zip(result, want[s]))


@pytest.mark.gpu
@pytest.mark.parametrize('m,n', [(8, 8), (20, 24), (20, 700), (300, 17), (64, 300), (50, 60)])
def test_orthogonalize_with_other_numbers_of_steps(m, n):
    """One step to many, also of matrices of lower rank, whose missing directions must not grow out of roundings: no singular value passes the quintic's
    largest, 1.2023.  Up to 8 steps also the value itself (later a rounding is multiplied by more than 1.5 in each step: the quintic at its fixed point)."""
    from boardlaw_amd import optim
    one, two = torch.ones((m, n), device='cuda'), gradient_like(m, 2, 'randn', 1).float() @ gradient_like(2, n, 'randn', 2).float()
    for g in (gradient_like(m, n, 'randn', 3).float(), gradient_like(m, n, 'decay', 4).float(), one, two):
        for steps in (1, 2, 3, 8, 9, 12, 16, 20, 40):
            out = optim.orthogonalize(g, steps=steps).double()
            assert torch.isfinite(out).all() and torch.linalg.matrix_norm(out, 2) <= 1.2023 * (1 + 1e-4), steps
            if steps <= 8:
                # A step adds a X, b A X and c A^2 X, where |X| and |A| go up to 1: a rounding of A counts 4.7750 times and twice 2.0315, one of A^2 2.0315,
                # of B X 4.7750 - 2.0315, of a X 3.4445: 17 in all, each of f32's size, or of 22 bits; times at most 3.4445 in each step behind it
                want = iteration(g, torch.float64, steps)
                assert (out - want).norm() <= 17 * U * steps * 3.4445 ** (steps - 1) * max(1., float(want.norm()))


@pytest.mark.gpu
@pytest.mark.parametrize('m,n', [(8, 8), (20, 24), (20, 700), (17, 300), (32, 16384), (64, 300), (4000, 8)])
def test_few_rows_of_lower_rank(m, n):
    """f64 on the m x m side, up to 6 steps: a rounding in A (products of up to 64 terms, two in a row: 16 at random) comes out 3.4445^3 = 41 times as
    large for each step behind it where the matrix lacks a direction, which is still f32's size."""
    from boardlaw_amd import optim
    row = gradient_like(1, n, 'randn', 5)
    mats = dict(ones=torch.ones((m, n), device='cuda'), same=row.expand(m, n), rank2=gradient_like(m, 2, 'randn', 1) @ gradient_like(2, n, 'randn', 2),
                one_row=torch.cat([row, torch.zeros((m - 1, n), device='cuda')]), steep=gradient_like(m, n, 'steep', 3))
    for name, g in mats.items():
        for steps in (1, 2, 3, 4, 5, 6):
            out, want = optim.orthogonalize(g.float(), steps=steps).double(), iteration(g.float(), torch.float64, steps)
            off = float((out - want).norm() / want.norm())
            assert off <= U + 16 * 2. ** -53 * 41. ** (steps - 1), (name, steps, off)
