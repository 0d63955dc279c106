"""The learner-step operators -- heads.logprobs, networks.norm_residual, optim.orthogonalize -- against plain implementations in 64 bits, at
the sizes, masks, strides and types where they can go wrong; their refusals; and a run of them together."""
import math

import numpy as np
import pytest
import torch

TYPES = [torch.float32, torch.float16, torch.bfloat16]
U = 2. ** -24                                       # half a step of f32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def close(got, want, tol, name=''):
    """|got - want| <= tol everywhere, infinities and NaN in the same places."""
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    tol = (tol.detach().double().cpu() if isinstance(tol, torch.Tensor) else torch.tensor(float(tol), dtype=torch.float64)).expand(want.shape)
    assert got.shape == want.shape, (name, got.shape, want.shape)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f'{name}: NaN in other places'
    assert torch.equal(got[~fine].nan_to_num(nan=0.), want[~fine].nan_to_num(nan=0.)), f'{name}: infinities in other places'
    off = (got - want).abs()[fine]
    assert (off <= tol[fine]).all(), f'{name}: {float((off / tol[fine].clamp_min(1e-300)).max()):.2f} of the tolerance'


# ---------------------------------------------------------------------------------------------------------------- logprobs

def plain_logprobs(raw, actions, valid, k):
    """heads.logprobs in 64 bits, with log p and what the tolerances need."""
    x = raw.detach().double()
    A = x.shape[-1]
    if valid is not None:
        x = torch.where(valid.expand(x.shape), x, -math.inf)
    some = (x > -math.inf).any(-1) | x.isnan().any(-1)
    m = torch.where(some, x.amax(-1), 0.)                           # (subtracted first: the lowest values keep their differences)
    logs = (x - m[..., None]).exp().sum(-1).log()
    logs = torch.where(m == math.inf, math.nan, torch.where(some, logs, 0.))
    lp = torch.where((x == -math.inf) & ~logs.isnan()[..., None], -math.inf, (x - m[..., None]) - logs[..., None])
    p = lp.exp()
    H = torch.where(p == 0, 0., -p * lp).sum(-1)
    out = dict(lp=lp, p=p, entropy=H, x=x)
    if actions is not None:
        a = actions.long()
        given = lp.gather(-1, a.clamp(0, A - 1)[..., None])[..., 0]
        out['logp'] = torch.where(a < 0, 0., torch.where(a >= A, math.nan, given))
    if k:
        order = torch.sort(x.nan_to_num(nan=math.inf, posinf=3e300, neginf=-math.inf), dim=-1, descending=True, stable=True).indices
        order = torch.nn.functional.pad(order[..., :k], (0, max(0, k - A)), value=0)
        real = (torch.arange(k, device=x.device) < A) & (x.gather(-1, order) != -math.inf)
        out['top'] = torch.where(real, order, -1)
        out['top_logp'] = torch.where(real, lp.gather(-1, order), -math.inf)
    return out


def plain_logprobs_grad(o, actions, g_logp, g_entropy, g_top):
    """The formula's gradient, and the sum of its terms' sizes."""
    lp, p, H = o['lp'], o['p'], o['entropy']
    A = lp.shape[-1]
    add, total = torch.zeros_like(lp), torch.zeros_like(H)
    if g_logp is not None:
        g = torch.where(actions < 0, 0., g_logp.double())
        add = add.scatter_add(-1, actions.long().clamp(0, A - 1)[..., None], g[..., None])
        total = total + g
    if g_top is not None:
        g = torch.where(o['top'] < 0, 0., g_top.double())
        add = add.scatter_add(-1, o['top'].clamp(min=0), g)
        total = total + g.sum(-1)
    gH = 0. if g_entropy is None else g_entropy.double()[..., None]
    l = torch.where(p == 0, 0., lp)
    live = o['x'] != -math.inf
    d = add - p * (total[..., None] + gH * (l + H[..., None]))
    size = add.abs() + p * (total.abs()[..., None] + abs(gH) * (l.abs() + H[..., None] + 2))
    return torch.where(live, d, 0.), torch.where(live, size, 0.)


def check_logprobs(raw, actions, valid, k, out):
    A = raw.shape[-1]
    w = plain_logprobs(raw, actions, valid, k)
    # the sum's roundings: a lane's share one after the other (A / 256, for the widest a 32nd of that again), joined over lanes, waves and
    # parts in under 20 steps of a few roundings; an exponential is |d| + 2 half steps off.  log s and x - m add one of their own size each
    terms = 48 + min(A, 1024) / 16 + A / 256
    spread = 2 + math.log(A)
    top = w['x'].nan_to_num(neginf=0.).abs().amax(-1)
    if actions is not None:
        close(out.logp, w['logp'], U * (terms + 3 * w['logp'].nan_to_num(neginf=0.).abs() + top), 'logp')
    close(out.entropy, w['entropy'], U * terms * spread, 'entropy')
    if k:
        assert torch.equal(out.top.cpu(), w['top'].cpu()), 'top'
        close(out.top_logp, w['top_logp'], U * (terms + 3 * w['top_logp'].nan_to_num(neginf=0.).abs() + top[..., None]), 'top_logp')
    return w


LOGPROBS = [(1, 1), (3, 2), (5, 16), (6, 33), (70, 81), (9, 97), (4, 169), (3, 256), (5, 257), (4, 513), (3, 1024), (3, 1025), (2, 5003), (600, 4100), (2, 32768), (1, 131071),
            (4099, 300), (4097, 512), (4098, 600), (4096, 1000), (2050, 1500)]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('R,A', LOGPROBS)
@pytest.mark.parametrize('masked', [False, True])
def test_logprobs(R, A, dtype, masked):
    from boardlaw_amd import heads
    gen = torch.Generator('cuda').manual_seed(R * A)
    raw = (3 * torch.randn((R, A), generator=gen, device='cuda')).to(dtype)
    actions = torch.randint(-1, A, (R,), generator=gen, device='cuda')
    valid = torch.rand((R, A), generator=gen, device='cuda') < .5 if masked else None
    for k in (0, 1, 5, 64):
        raw.requires_grad_()
        out = heads.logprobs(raw, actions, valid, k)
        w = check_logprobs(raw, actions, valid, k, out)
        size = 64. if dtype == torch.float16 else 1.
        gs = [size * torch.randn(o.shape, generator=gen, device='cuda') for o in (out.logp, out.entropy)]
        outs = [out.logp, out.entropy]
        if k:
            gs.append(size * torch.randn((R, k), generator=gen, device='cuda')); outs.append(out.top_logp)
        d, = torch.autograd.grad(outs, raw, gs, retain_graph=True)
        with pytest.raises(RuntimeError, match='differentiable once'):
            torch.autograd.grad(outs, raw, gs, create_graph=True)
        want, mag = plain_logprobs_grad(w, actions, gs[0], gs[1], gs[2] if k else None)
        assert d.dtype == dtype
        # p is as exact as logp; a sum of k gradients adds k roundings; one to the result's type (in f16 also of the smallest steps)
        terms = 64 + min(A, 1024) / 16 + A / 256 + k + 4 * w['lp'].nan_to_num(neginf=0.).abs() + w['x'].nan_to_num(neginf=0.).abs().amax(-1, keepdim=True)
        total = sum(g.abs().reshape(R, -1).sum(-1, keepdim=True) for g in gs).double()
        close(d, want, U * terms * (mag + w['p'] * total) + half_step(dtype) * want.abs() + torch.finfo(dtype).tiny * half_step(dtype) * 2 + 1e-38, 'd_raw')
        raw = raw.detach()
        # without a gradient the same numbers
        again = heads.logprobs(raw, actions, valid, k)
        assert torch.equal(again.entropy, out.entropy) and torch.equal(again.logp, out.logp)


@pytest.mark.gpu
@pytest.mark.parametrize('A', [6, 81, 700, 9001])
@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_logprobs_borders(A, dtype):
    """Rows without a valid move, with one, with the type's lowest value, -inf, +inf and NaN, in valid and in masked places; moves that are invalid,
    missing or beyond the row; ties."""
    from boardlaw_amd import heads
    low = torch.finfo(dtype).min
    raw = torch.randn((12, A), device='cuda').to(dtype)
    valid = torch.rand((12, A), device='cuda') < .7
    valid[:, :4] = True
    actions = torch.zeros(12, dtype=torch.int32, device='cuda')
    valid[0] = False                                                # nothing
    valid[1] = False; valid[1, A - 1] = True; actions[1] = A - 1    # one move
    raw[2] = low                                                    # the lowest value is a value
    raw[3] = -math.inf                                              # nothing, by the logits
    raw[4, 1] = -math.inf; actions[4] = 1                           # an impossible move given
    valid[5, 2] = False; raw[5, 2] = math.nan; valid[5, 3] = False; raw[5, 3] = math.inf; actions[5] = 2      # masked places hold anything
    raw[6, 1] = math.nan
    raw[7, 3] = math.inf
    raw[8] = 0.; raw[8, ::2] = -0.; actions[8] = -1                 # ties, of both zeros; no move
    actions[9] = A
    raw[10, 1:3] = raw[10].max() + 1                                # two best
    raw[11] = low; raw[11, 0] = 8.
    raw.requires_grad_()
    out = heads.logprobs(raw, actions, valid, k=5)
    w = plain_logprobs(raw, actions, valid, 5)
    w['x'] = w['x'].nan_to_num(nan=0., posinf=0.)
    fine = torch.tensor([0, 1, 2, 3, 4, 5, 8, 10, 11], device='cuda')
    check_logprobs(raw[fine], actions[fine], valid[fine], 5, type(out)((k, v[fine]) for k, v in out.items()))
    assert out.entropy[[0, 3]].tolist() == [0, 0] and out.logp[[0, 3]].tolist() == [-math.inf] * 2 and (out.top[[0, 3]] == -1).all()
    assert out.logp[4] == -math.inf and out.logp[5] == -math.inf and out.logp[8] == 0 and out.logp[9].isnan() and not out.entropy[9].isnan()
    assert out.entropy[[6, 7]].isnan().all() and out.logp[[6, 7]].isnan().all() and out.top_logp[[6, 7], 0].isnan().all()
    assert out.top[6, 0] == 1 and out.top[7, 0] == 3
    assert out.top[8].tolist() == (torch.nonzero(valid[8])[:5, 0].tolist() + [-1] * 5)[:5]
    assert set(out.top[10, :2].tolist()) == {1, 2} and out.top[10, 0] == 1
    assert out.logp[1] == 0 and out.entropy[1] == 0
    d, = torch.autograd.grad([out.logp, out.entropy], raw, [torch.ones_like(out.logp), torch.ones_like(out.entropy)])
    assert (d[[0, 3]] == 0).all() and (d[~valid] == 0).all()
    assert d[1, A - 1] == 0 and d[6, 0].isnan() and d[9, 0].isnan()
    rest = [2, 4, 5, 8, 10, 11]
    assert torch.isfinite(d[rest]).all()


@pytest.mark.gpu
def test_logprobs_keeps_the_rest_of_a_sure_row():
    """One move with nearly all the mass: its logp and the entropy are the rest's mass, far below 1's rounding."""
    from boardlaw_amd import heads
    for A in (81, 600, 5000):
        raw = torch.full((3, A), -30., device='cuda', dtype=torch.float32)
        raw[:, 7] = 0.
        out = heads.logprobs(raw, torch.full((3,), 7, device='cuda'), k=1)
        r = (A - 1) * math.exp(-30)
        assert np.allclose(out.logp.cpu().double(), -math.log1p(r), rtol=64 * U, atol=0)
        assert np.allclose(out.entropy.cpu().double(), math.log1p(r) + 30 * r / (1 + r), rtol=64 * U, atol=0)


@pytest.mark.gpu
@pytest.mark.parametrize('A', [81, 1024, 4099, 8192])
@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_logprobs_layouts(A, dtype):
    """Views: rows of a wider tensor, from an odd column, transposed, expanded; (T, B, A) leading dims; one mask for all rows; whole numbers of any type."""
    from boardlaw_amd import heads
    base = torch.randn((7, A + 24), device='cuda').to(dtype)
    mask = torch.rand((A,), device='cuda') < .8
    mask[:8] = True
    wide = torch.rand((7, A + 24), device='cuda') < .8
    for raw in (base[:, 8:8 + A], base[:, 3:3 + A], base[:, :A].T.contiguous().T, base[:1, :A].expand(5, A), base[:6, 8:8 + A].unflatten(0, (3, 2))):
        lead = raw.shape[:-1]
        for valid in (None, mask, mask.expand(raw.shape), wide[:lead.numel(), 1:1 + A].reshape(raw.shape) if raw.ndim == 3 else wide[:lead.numel(), 1:1 + A]):
            actions = torch.randint(0, 8, lead, device='cuda', dtype=torch.int16)
            x = raw.detach().requires_grad_()
            out = heads.logprobs(x, actions, valid, k=3)
            w = check_logprobs(raw, actions, valid, 3, out)
            g = torch.randn(lead, device='cuda')
            d, = torch.autograd.grad(out.logp, x, g)
            want, mag = plain_logprobs_grad(w, actions.long(), g, None, None)
            terms = 64 + min(A, 1024) / 16 + A / 256 + 4 * w['lp'].nan_to_num(neginf=0.).abs() + 4
            close(d, want, U * terms * mag + half_step(dtype) * want.abs() + torch.finfo(dtype).tiny * half_step(dtype) * 2 + 1e-38, 'd_raw')
    assert heads.logprobs(base[:0, :A], None, None, 2).top.shape == (0, 2)


@pytest.mark.gpu
@pytest.mark.parametrize('A', [81, 2000])
def test_logprobs_gradient_against_differences(A):
    from boardlaw_amd import heads
    torch.manual_seed(A)
    raw = torch.randn((4, A), device='cuda').requires_grad_()
    actions = torch.randint(0, A, (4,), device='cuda')
    v = torch.randn((4, A), device='cuda')

    def f(x):
        o = heads.logprobs(x, actions, None, 3)
        return (o.logp + 2 * o.entropy + 3 * o.top_logp.sum(-1)).double()

    g, = torch.autograd.grad(f(raw).sum(), raw)
    h = 2. ** -7
    num = (f(raw.detach() + h * v) - f(raw.detach() - h * v)) / (2 * h)
    # f's rounding (values to 60, ~100 half steps) over h; the cubic term: third derivatives of a log-sum-exp are under 4 |v|^3 p-weighted
    assert ((g.double() * v.double()).sum(-1) - num).abs().max() <= 60 * 100 * U / h + h * h * 12 * 30


# ------------------------------------------------------------------------------------------------------------ norm_residual

def plain_norm(x, y, alpha, post, gate, pre, eps):
    """networks.norm_residual in 64 bits, by autograd over elementary operations."""
    W = x.shape[-1]
    x = x.double()
    if y is None:
        return None, pre.double() * x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    y = y.double()
    if y.shape[-1] == 2 * W:
        y, gate = y[..., :W], y[..., W:]
    n = y
    if post is not None:
        n = post.double() * y / (y.square().mean(-1, keepdim=True) + eps).sqrt()
    if gate is not None:
        n = torch.sigmoid(gate.double()) * n
    out = x + (1. if alpha is None else alpha.double()) * n
    return out, None if pre is None else pre.double() * out / (out.square().mean(-1, keepdim=True) + eps).sqrt()


NORMS = [(1, 1), (3, 2), (3, 7), (5, 16), (9, 100), (37, 128), (3, 129), (130, 512), (2, 771), (3, 1024), (5, 2048), (2, 2049), (3, 4104), (2, 8191), (2, 8192)]
PAIRS = [(torch.float32, torch.float32), (torch.float32, torch.float16), (torch.float32, torch.bfloat16), (torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16)]


def norm_inputs(R, W, tx, ty, gate, seed=0):
    g = torch.Generator('cuda').manual_seed(seed + R * W)
    n = lambda *s: torch.randn(s, generator=g, device='cuda')
    y = n(R, 2 * W if gate == 'packed' else W).to(ty)
    gates = dict(none=None, packed=None, full=n(R, W).to(ty), channel=n(W), row=n(R, 1).to(ty))
    return dict(x=n(R, W).to(tx), y=y, alpha=torch.tensor(0.6, device='cuda'), post=1 + .2 * n(W), gate=gates[gate], pre=1 + .2 * n(W)), n


def check_norm(t, out, h, grads, g_out, g_h, eps=1e-5):
    names = [k for k, v in t.items() if v is not None]
    leaves = {k: t[k].detach().double().requires_grad_() for k in names}
    wo, wh = plain_norm(*[leaves.get(k) for k in ('x', 'y', 'alpha', 'post', 'gate', 'pre')], eps)
    W = t['x'].shape[-1]
    # a row's sum of W squares in lanes of 8, joined: under 8 + W / 64 / 8 + 8 roundings, halved by the root; the products a few more
    k = 24 + W / 512
    if out is not None:
        close(out, wo, half_step(out.dtype) * wo.abs() + U * k * (1 + wo.abs() + (wo - leaves['x']).abs()) + torch.finfo(out.dtype).tiny * half_step(out.dtype) * 2, 'x_out')
    if h is not None:
        # x_out's cancellation, seen through 1 / rms
        scale = wh.abs() + ((wo.detach().abs() + leaves['x'].abs()) if wo is not None else leaves['x'].abs()) * (t['pre'].abs().double() / ((wo if wo is not None else leaves['x']).square().mean(-1, keepdim=True) + eps).sqrt())
        close(h, wh, half_step(h.dtype) * wh.abs() + 2 * U * k * scale + torch.finfo(h.dtype).tiny * half_step(h.dtype) * 2, 'h')
    if grads is None:
        return
    given = [(o, g.double()) for o, g in ((wo, g_out), (wh, g_h)) if g is not None]
    want = torch.autograd.grad([o for o, _ in given], list(leaves.values()), [g for _, g in given], allow_unused=True)
    for name, got, w in zip(names, grads, want):
        w = torch.zeros_like(leaves[name]) if w is None else w
        R = t['x'].shape[0]
        # sums over rows add roundings of their own: a lane's rows, 4 or 16 groups, the workgroups' sums in four parts
        rows = 0 if name in ('x', 'y') else 8 + min(R, 256)
        # against the size of what is summed, which the row's (column's) largest stand for; the reciprocal rms (1 / sqrt(eps) at most) scales y's and x's
        rms = w.square().mean().sqrt() + w.abs().amax() * 1.
        close(got, w, half_step(got.dtype) * w.abs() + U * (4 * k + rows) * rms * 4 + torch.finfo(got.dtype).tiny * half_step(got.dtype) * 2, f'd_{name}')


@pytest.mark.gpu
@pytest.mark.parametrize('tx,ty', PAIRS, ids=str)
@pytest.mark.parametrize('R,W', NORMS)
def test_norm_residual(R, W, tx, ty):
    from boardlaw_amd import networks
    for gate in ('none', 'packed', 'full', 'channel', 'row'):
        t, n = norm_inputs(R, W, tx, ty, gate)
        leaves = [v.requires_grad_() for v in t.values() if v is not None]
        out, h = networks.norm_residual(**t)
        assert out.dtype == tx and h.dtype == ty
        g_out, g_h = n(R, W).to(tx), n(R, W).to(ty)
        # a zero-mean sum over rows can come out near 0: lean it
        g_out = (g_out.float() + t['y'][:, :W].detach().float()).to(tx)
        grads = torch.autograd.grad([out, h], leaves, [g_out, g_h])
        assert all(a.shape == b.shape and a.dtype == b.dtype for a, b in zip(grads, leaves))
        check_norm({k: None if v is None else v.detach() for k, v in t.items()}, out, h, grads, g_out, g_h)
        with torch.no_grad():
            o2, h2 = networks.norm_residual(**t)
        assert torch.equal(o2, out) and torch.equal(h2, h)


@pytest.mark.gpu
@pytest.mark.parametrize('W', [40, 100, 513, 3000])
def test_norm_residual_parts(W):
    """Without each of the optional pieces; one output's gradient only; rows of wider tensors; (T, B, W); no rows."""
    from boardlaw_amd import networks
    R = 11
    base, n = norm_inputs(R, W, torch.float32, torch.float16, 'full')
    for drop in ((), ('alpha',), ('post',), ('pre',), ('gate', 'post'), ('alpha', 'post', 'gate')):
        for only in ('both', 'out', 'h'):
            if only == 'h' and 'pre' in drop:
                continue
            t = {k: None if k in drop else v.detach().requires_grad_() for k, v in base.items()}
            out, h = networks.norm_residual(**t, eps=1e-3)
            assert (h is None) == ('pre' in drop)
            g_out = n(R, W) if only != 'h' else None
            g_h = n(R, W).half() if only != 'out' and h is not None else None
            leaves = [v for v in t.values() if v is not None]
            pairs = [(o, g) for o, g in ((out, g_out), (h, g_h)) if g is not None]
            grads = torch.autograd.grad([o for o, _ in pairs], leaves, [g for _, g in pairs], allow_unused=True)
            grads = [torch.zeros_like(l) if g is None else g for g, l in zip(grads, leaves)]
            check_norm({k: None if v is None else v.detach() for k, v in t.items()}, out, h, grads, g_out, g_h, 1e-3)
    # only the norm before
    x = n(R, W).requires_grad_()
    pre = (1 + n(W)).requires_grad_()
    same, h = networks.norm_residual(x, pre=pre, dtype=torch.bfloat16)
    assert same is x and h.dtype == torch.bfloat16
    g = n(R, W).bfloat16()
    grads = torch.autograd.grad(h, [x, pre], g)
    check_norm(dict(x=x.detach(), y=None, alpha=None, post=None, gate=None, pre=pre.detach()), None, h, grads, None, g)
    # layouts
    wide = n(R, 3 * W + 8)
    for lo in (0, 8, 3):
        t = dict(x=wide[:, lo:lo + W], y=wide[:, W:2 * W], alpha=None, post=base['post'].detach(), gate=wide[:, 2 * W - lo:3 * W - lo], pre=base['pre'].detach())
        check_norm(t, *networks.norm_residual(**t), None, None, None)
        check_norm(dict(t, x=t['x'].T.contiguous().T), *networks.norm_residual(**dict(t, x=t['x'].T.contiguous().T)), None, None, None)
    x3, y3 = n(2, 5, W), n(2, 5, 2 * W)
    o3, h3 = networks.norm_residual(x3, y3, pre=base['pre'])
    assert torch.equal(o3.view(10, W), networks.norm_residual(x3.view(10, W), y3.view(10, 2 * W), pre=base['pre'])[0]) and h3.shape == x3.shape
    x0 = torch.empty((0, W), device='cuda', requires_grad=True)
    p0 = base['pre'].detach().requires_grad_()
    o0, h0 = networks.norm_residual(x0, x0, pre=p0)
    gx, gp = torch.autograd.grad(h0.sum(), [x0, p0])
    assert gx.shape == (0, W) and (gp == 0).all()


@pytest.mark.gpu
def test_norm_residual_borders():
    """Rows of zeros and of ones that differ by 1e4, gates at both ends and at infinity, NaN only in its own row."""
    from boardlaw_amd import networks
    W = 64
    x, y, gate = torch.randn((6, W), device='cuda'), torch.randn((6, W), device='cuda'), torch.randn((6, W), device='cuda')
    post, pre = torch.ones(W, device='cuda'), torch.ones(W, device='cuda')
    x[0] = 0; y[0] = 0
    y[1] *= 1e4; x[1] *= 1e-4
    gate[2] = -math.inf; gate[3] = math.inf; gate[4, ::2] = -200.; gate[4, 1::2] = 200.
    y[5, 3] = math.nan
    ts = [v.requires_grad_() for v in (x, y, gate)]
    out, h = networks.norm_residual(x, y, None, post, gate, pre)
    wo, wh = plain_norm(x, y, None, post, gate, pre, 1e-5)
    close(out[:5], wo[:5], U * 40 * (wo[:5].abs() + 1))
    close(h[:5], wh[:5], U * 60 * (wh[:5].abs() + 1))
    assert out[5].isnan().all() and h[5].isnan().all()
    d = torch.autograd.grad([out[:5].sum(), h[:5].sum()], ts, allow_unused=True)
    assert all(torch.isfinite(t[:5]).all() for t in d)
    assert (d[2][2:5] == 0).all() and (d[1][2] == 0).all()


@pytest.mark.gpu
def test_norm_residual_gradient_against_differences():
    from boardlaw_amd import networks
    t, n = norm_inputs(6, 50, torch.float32, torch.float32, 'full')
    a, b = n(6, 50), n(6, 50)
    f = lambda t: sum((o.double() * w.double()).sum() for o, w in zip(networks.norm_residual(**t), (a, b)))
    leaves = {k: v.requires_grad_() for k, v in t.items()}
    grads = dict(zip(leaves, torch.autograd.grad(f(leaves), list(leaves.values()))))
    for name in leaves:
        v = n(*leaves[name].shape) if leaves[name].ndim else torch.ones((), device='cuda')
        h = 2. ** -8
        num = (f({**t, name: (t[name] + h * v).detach()}) - f({**t, name: (t[name] - h * v).detach()})) / (2 * h)
        # f sums 600 products of size about 1, each 30 half steps off at random, over h; cubic terms of 600 elements at h^2 (coefficients under 3)
        assert abs((grads[name].double() * v.double()).sum() - num) <= 30 * U * 600 ** .5 * 8 / h + h * h * 3 * 600, name


# ------------------------------------------------------------------------------------------------------------ orthogonalize

def plain_ortho(g, steps=5, eps=1e-7):
    x = g.double()
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    x = x / (x.norm() + eps)
    for _ in range(steps):
        a = x @ x.T
        x = 3.4445 * x + (-4.7750 * a + 2.0315 * a @ a) @ x
    return x.T if tall else x


def spectrum(m, n, lo, seed):
    """A matrix of Frobenius norm 3 whose singular values lie between lo and 1 of the largest."""
    g = torch.Generator().manual_seed(seed)
    q = min(m, n)
    u, _ = torch.linalg.qr(torch.randn((m, q), generator=g, dtype=torch.float64))
    v, _ = torch.linalg.qr(torch.randn((n, q), generator=g, dtype=torch.float64))
    s = torch.logspace(math.log10(lo), 0, q, dtype=torch.float64) if q > 1 else torch.ones(1, dtype=torch.float64)
    x = (u * s) @ v.T
    return 3 * x / x.norm()


ORTHO = [(1, 1), (1, 7), (9, 1), (16, 16), (20, 33), (64, 64), (65, 64), (63, 130), (128, 128), (129, 127), (162, 512), (300, 100), (512, 512), (770, 257)]


def ortho_tolerance(dtype, want, steps=5):
    # operands are 2^-22 off (entries), sums of k products add sqrt(k) 2^-24 at random, and a direction's error is multiplied by 3.4445 in each step
    # that follows, at most: 3.4445^4 for the first product's.  In the norm of the whole
    size = want.double().norm()
    return size * (steps * 4 * 2. ** -22) * 3.4445 ** (steps - 1)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('m,n', ORTHO)
def test_orthogonalize(m, n, dtype):
    from boardlaw_amd import optim
    mats = [spectrum(m, n, lo, i).to(dtype).cuda() for i, lo in enumerate((.5, .02, .5))]
    outs = optim.orthogonalize(mats)
    for i, (g, o) in enumerate(zip(mats, outs)):
        want = plain_ortho(g.cpu())
        assert o.shape == g.shape and o.dtype == dtype
        off = (o.cpu().double() - want).norm()
        assert off <= ortho_tolerance(dtype, want) + half_step(dtype) * want.norm(), (i, float(off / want.norm()))
        s = torch.linalg.svdvals(want)
        assert s.max() < 1.25
    assert torch.equal(outs[0], optim.orthogonalize(mats[:1])[0]), 'a matrix does not depend on its batch'
    assert all(torch.equal(a, b) for a, b in zip(optim.orthogonalize(torch.stack(mats)), outs))


@pytest.mark.gpu
@pytest.mark.parametrize('count,m,n', [(1, 64, 128), (2, 128, 64), (33, 50, 100), (9, 512, 512), (20, 512, 512), (8, 1024, 1024), (7, 700, 900), (6, 1030, 500), (1, 2048, 2048)])
def test_orthogonalize_many(count, m, n):
    """Batches that take each of the products' tilings, against 64 bits on the device; twice the same."""
    from boardlaw_amd import optim
    gen = torch.Generator('cuda').manual_seed(m)
    mats = [torch.randn((m, n), generator=gen, device='cuda') for _ in range(count)]
    outs = optim.orthogonalize(mats)
    for g, o in zip(mats, outs):
        want = plain_ortho(g)
        assert (o.double() - want).norm() <= ortho_tolerance(torch.float32, want)
        assert (o.double() - want).abs().max() <= ortho_tolerance(torch.float32, want)
    assert all(torch.equal(a, b) for a, b in zip(outs, optim.orthogonalize(mats)))


@pytest.mark.gpu
def test_orthogonalize_borders():
    """Zero, rank one, scales from 1e-30 to 1e30, a list of several shapes and types, views, NaN in one matrix only, more matrices than one launch takes,
    nothing."""
    from boardlaw_amd import optim
    z, one, nan = torch.zeros((40, 24), device='cuda'), torch.ones((40, 24), device='cuda'), torch.full((40, 24), math.nan, device='cuda')
    oz, o1, on = optim.orthogonalize([z, one, nan])
    assert (oz == 0).all() and on.isnan().all()
    want = plain_ortho(one.cpu())
    assert (o1.cpu() - want).norm() <= ortho_tolerance(torch.float32, want)
    g = spectrum(48, 70, .3, 0).float().cuda()
    base = optim.orthogonalize(g)
    for scale in (2. ** -100, 2. ** 100):
        assert torch.equal(optim.orthogonalize([g * scale], eps=0.)[0], optim.orthogonalize([g], eps=0.)[0])
    mixed = [g, spectrum(30, 10, .5, 1).half().cuda(), spectrum(48, 70, .3, 2).float().cuda(), g[:, 3:40], g.T]
    outs = optim.orthogonalize(mixed)
    assert torch.equal(outs[0], base)
    for a, b in zip(mixed, outs):
        assert a.dtype == b.dtype and a.shape == b.shape
        want = plain_ortho(a.cpu())
        assert (b.cpu().double() - want).norm() <= ortho_tolerance(a.dtype, want) + half_step(a.dtype) * want.norm()
    many = [spectrum(20, 12, .5, i).float().cuda() for i in range(37)]
    for a, b in zip(many, optim.orthogonalize(many)):
        assert torch.equal(b, optim.orthogonalize(a))
    assert optim.orthogonalize([]) == [] and optim.orthogonalize(torch.zeros((0, 3, 4), device='cuda')).shape == (0, 3, 4)
    for steps in (1, 2, 8):
        want = plain_ortho(g.cpu(), steps)
        assert (optim.orthogonalize(g, steps=steps).cpu() - want).norm() <= ortho_tolerance(torch.float32, want, min(steps, 5))


@pytest.mark.gpu
def test_muon_is_its_formula():
    from boardlaw_amd import optim
    torch.manual_seed(0)
    shapes = [(48, 48), (96, 48), (48, 48), (48, 96)]
    ps = [torch.nn.Parameter(torch.randn(s, device='cuda')) for s in shapes]
    ref = [p.detach().double().cpu() for p in ps]
    ms = [torch.zeros(s, dtype=torch.float64) for s in shapes]
    opt = optim.Muon(ps, lr=.05, momentum=.9, weight_decay=.1)
    for step in range(3):
        for i, p in enumerate(ps):
            p.grad = spectrum(*p.shape, .3, 10 * step + i).float().cuda()
        opt.step()
        for i, p in enumerate(ps):
            g = p.grad.double().cpu()
            ms[i] = .9 * ms[i] + g
            ref[i] = (1 - .05 * .1) * ref[i] - .05 * max(1, p.shape[0] / p.shape[1]) ** .5 * plain_ortho(g + .9 * ms[i])
            # each step: a few roundings of the weights, and lr times the update's error (with its inputs' roundings)
            assert (p.detach().cpu().double() - ref[i]).norm() <= (step + 1) * (4 * U * ref[i].norm() + .05 * 1.5 * 2 * ortho_tolerance(torch.float32, ref[i] / ref[i].norm() * 7))
    other = optim.Muon(ps)
    other.load_state_dict(opt.state_dict())
    assert torch.equal(other.state[ps[0]]['momentum'], opt.state[ps[0]]['momentum'])


# ---------------------------------------------------------------------------------------------- streams, graphs, together

@pytest.mark.gpu
def test_operators_on_streams_and_in_graphs():
    """Two streams at once give what one gives; a captured step replayed on new inputs gives the eager results, every time, also between eager calls."""
    from boardlaw_amd import heads, networks, optim
    W, A, R = 256, 5000, 8

    def make(seed):
        g = torch.Generator('cuda').manual_seed(seed)
        n = lambda *s: torch.randn(s, generator=g, device='cuda')
        return [n(R, A), n(300, W), n(300, 2 * W).half(), n(W), n(W), n(200, 90)]

    def step(t):
        raw, x, y, post, pre, g = t
        raw, x = raw.detach().requires_grad_(), x.detach().requires_grad_()
        post, pre = post.detach().requires_grad_(), pre.detach().requires_grad_()
        o = heads.logprobs(raw, torch.arange(R, device='cuda'), raw > -2, k=4)
        xo, h = networks.norm_residual(x, y, None, post, pre=pre)
        d = torch.autograd.grad([o.logp.sum() + o.entropy.sum(), xo.sum(), h.float().square().sum()], [raw, x, post, pre])
        return [o.logp, o.entropy, o.top, o.top_logp, xo, h, *d, optim.orthogonalize(g)]

    want = {s: [t.clone() for t in step(make(s))] for s in range(4)}
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = {}
    for s in range(4):
        with torch.cuda.stream(streams[s % 2]):
            got[s] = step(make(s))
    torch.cuda.synchronize()
    for s in range(4):
        assert all(torch.equal(a, b) for a, b in zip(got[s], want[s]))
    graphs = []
    for _ in range(2):
        static = make(0)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(static)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(static)
        graphs.append((graph, static, outs))
    for s in (1, 2, 3, 1):
        for graph, static, outs in graphs:
            for dst, src in zip(static, make(s)):
                dst.copy_(src)
            graph.replay()
            step(make(0))
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, want[s])), s


@pytest.mark.gpu
@pytest.mark.parametrize('block', ['rezero', 'gated'])
def test_a_learner_with_all_of_them(block):
    """training.run: self-play with the network's inference plan, entropy bonus, Muon for the blocks -- weights move and stay finite; the checkpoint comes back;
    the plans agree with the module."""
    import io
    from boardlaw_amd import hex, networks, storage, training
    torch.manual_seed(0)
    worlds = hex.Hex.initial(32, 5)
    net = networks.FCModel(worlds.obs_space, worlds.action_space, width=128, depth=3, block=block).cuda()
    before = {k: v.clone() for k, v in net.state_dict().items()}
    seen = []
    training.run(worlds, net, n_steps=3, nodes=8, buffer_len=4, inference='fused', graph=True, optimizer='muon', hidden_lr=.01, entropy=.05, on_step=lambda s, p, v: seen.append((float(p), float(v))))
    after = net.state_dict()
    assert len(seen) == 3 and np.isfinite(seen).all()
    assert all(torch.isfinite(v).all() for v in after.values())
    moved = [k for k in after if not torch.equal(after[k], before[k])]
    assert 'body.2.weight' in moved and 'body.1.α' in moved and 'policy.core.weight' in moved
    if block == 'gated':
        assert 'body.1.post' in moved and 'body.2.pre' in moved
    twin = storage.network_from_state({'network.' + k: v for k, v in after.items()}, 'cuda')
    assert type(twin.body) is type(net.body)
    w = hex.Hex.initial(16, 5)
    a, b = net(w), twin(w)
    assert torch.equal(a.logits, b.logits) and torch.equal(a.v, b.v)
    plan = networks.Inference(net, fused=True)
    p32, v32 = plan.root_raw(w)
    p, v = net.raw(w)
    # two GEMM orders of f32: 128 to 512 products of size under 1, random
    assert (p32 - p).abs().max() <= 1e-4 and (v32 - v).abs().max() <= 1e-4
    w.obs_f16 = None
    p16, v16 = plan.raw(w)
    # f16 weights and branches, four Linears deep: 2^-11 of the neck's size each
    assert (p16.float() - p).abs().max() <= 8 * 2 ** -11 * (1 + p.abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize('precision', ['fp16', 'fp32'])
def test_gated_network_in_a_search(precision):
    """A search on a gated network's inference plan, eager and captured: the same moves; a plan follows its module's weights."""
    from boardlaw_amd import hex, networks
    from boardlaw_amd.mcts import MCTSAgent
    worlds = hex.Hex.initial(16, 4)
    torch.manual_seed(1)
    net = networks.FCModel(worlds.obs_space, worlds.action_space, width=40, depth=2, block='gated').cuda()
    with torch.no_grad():
        for b in list(net.body)[1:]:
            getattr(b, 'α').fill_(.5)
    plan = networks.Inference(net, precision=precision)
    seen = []
    for graph in (False, True):
        agent = MCTSAgent(plan, n_nodes=8, graph=graph)
        agent(worlds)
        torch.manual_seed(3)
        seen.append(agent(worlds))
    assert torch.equal(seen[0].actions, seen[1].actions) and torch.equal(seen[0].logits, seen[1].logits)
    before = plan.root_raw(worlds)[0].clone()
    with torch.no_grad():
        net.body[1].post.mul_(2.)
    assert not torch.equal(before, plan.root_raw(worlds)[0])


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """Tensors of more than 2^31 elements: their last rows are computed and written where they are."""
    from boardlaw_amd import heads, networks
    R, A = 70000, 32768
    raw = torch.zeros((R, A), dtype=torch.bfloat16, device='cuda')
    raw[-3:] = torch.randn((3, A), device='cuda').bfloat16()
    actions = torch.full((R,), A - 1, device='cuda')
    tail = raw[-3:].clone().requires_grad_()
    want = heads.logprobs(tail, actions[-3:], k=3)
    raw.requires_grad_()
    got = heads.logprobs(raw, actions, k=3)
    # (another number of waves per row: other roundings)
    assert torch.equal(got.top[-3:], want.top) and torch.allclose(got.entropy[-3:], want.entropy, rtol=200 * U) and torch.allclose(got.logp[-3:], want.logp, rtol=200 * U)
    # equal entries: c of them and nothing else, log s one rounding of log A off
    assert torch.allclose(got.entropy[:-3].double(), torch.full((), math.log(A), dtype=torch.float64, device='cuda'), rtol=4 * U, atol=0)
    d, = torch.autograd.grad(got.logp.sum(), raw)
    e, = torch.autograd.grad(want.logp.sum(), tail)
    assert torch.allclose(d[-3:].float(), e.float(), rtol=4 * half_step(torch.bfloat16), atol=1e-12)
    assert (d[::9000, -1] > .9).all()
    del raw, got, d
    R, W = 270000, 8192
    x = torch.zeros((R, W), dtype=torch.float16, device='cuda')
    x[-2:] = torch.randn((2, W), device='cuda').half()
    pre = torch.rand(W, device='cuda')
    out, h = networks.norm_residual(x, x, None, pre, None, pre)
    o2, h2 = networks.norm_residual(x[-2:].clone(), x[-2:].clone(), None, pre, None, pre)
    assert torch.equal(out[-2:], o2) and torch.equal(h[-2:], h2) and (out[:4] == 0).all() and (h[R - 3] == 0).all()


@pytest.mark.gpu
def test_single_rows():
    """One row without leading dimensions."""
    from boardlaw_amd import heads, networks
    x = torch.randn(81, device='cuda')
    out = heads.logprobs(x, torch.tensor(3, device='cuda'), x > 0, k=2)
    two = heads.logprobs(x[None], torch.tensor([3], device='cuda'), (x > 0)[None], k=2)
    assert out.logp.shape == () and out.top.shape == (2,) and all(torch.equal(a, b[0]) for a, b in zip(out.values(), two.values()))
    y, w = torch.randn(162, device='cuda'), torch.ones(81, device='cuda')
    a, b = networks.norm_residual(x, y, None, w, pre=w), networks.norm_residual(x[None], y[None], None, w, pre=w)
    assert a[0].shape == a[1].shape == (81,) and torch.equal(a[0], b[0][0]) and torch.equal(a[1], b[1][0])


@pytest.mark.gpu
def test_head_evaluates_without_the_rows():
    from boardlaw_amd import heads
    torch.manual_seed(0)
    head = heads.MaskedOutput(heads.Masked(81), 64).cuda()
    x = torch.randn((50, 64), device='cuda')
    valid = torch.rand((50, 81), device='cuda') < .5
    valid[:, 0] = True
    logits = head(x, valid)
    out = head.evaluate(x, valid, torch.zeros(50, dtype=torch.int64, device='cuda'), k=2)
    # two f32 log-softmaxes of the same raw rows
    assert (out.logp - logits[:, 0]).abs().max() <= 32 * U * 16
    assert torch.equal(out.top[:, 0], logits.argmax(-1))


# ---------------------------------------------------------------------------------------------------------------- refusals

def test_refusals():
    """Bad arguments end in an error before anything is launched (CPU tensors: shapes and types first, then the device)."""
    from boardlaw_amd import _native, heads, networks, optim, training
    z = torch.zeros
    with pytest.raises(_native.NativeError, match='no CPU fallback'):
        heads.logprobs(z(3, 4))
    with pytest.raises(TypeError):
        heads.logprobs(z(3, 4, dtype=torch.float64))
    with pytest.raises(ValueError):
        heads.logprobs(z(3, 0))
    with pytest.raises(ValueError):
        heads.logprobs(z(3, 4), k=65)
    with pytest.raises(_native.NativeError):
        networks.norm_residual(z(3, 4), z(3, 4), pre=z(4))
    with pytest.raises(ValueError):
        networks.norm_residual(z(3, 8193), pre=z(8193))
    with pytest.raises(TypeError):
        networks.norm_residual(z(3, 4, dtype=torch.float64), pre=z(4))
    with pytest.raises(_native.NativeError):
        optim.orthogonalize(z(3, 4))
    with pytest.raises(ValueError):
        optim.orthogonalize(z(4))
    with pytest.raises(TypeError):
        optim.orthogonalize([z(3, 4, dtype=torch.float64)])
    with pytest.raises(ValueError):
        optim.orthogonalize([z(1, 16385)])
    for steps, error in ((0, ValueError), (-1, ValueError), (1001, ValueError), (2.5, TypeError)):
        with pytest.raises(error):
            optim.orthogonalize(z(3, 4), steps=steps)
    with pytest.raises(ValueError):
        optim.Muon([torch.nn.Parameter(z(3))])
    with pytest.raises(ValueError):
        networks.FCModel(heads.Tensor((3, 3, 2)), heads.Masked(9), width=16, depth=2, block='other')
    net = networks.FCModel(heads.Tensor((3, 3, 2)), heads.Masked(9), width=16, depth=2)
    with pytest.raises(ValueError):
        training.make_optimizer(net, 'sgd')
    muon, adam = training.make_optimizer(net, 'muon')
    assert {id(p) for o in (muon, adam) for g in o.param_groups for p in g['params']} == {id(p) for p in net.parameters()}
    assert [tuple(p.shape) for p in muon.param_groups[0]['params']] == [(16, 16)] * 2


def test_several_optimisers_are_saved_as_one(tmp_path):
    from boardlaw_amd import heads, networks, storage, training
    net = networks.FCModel(heads.Tensor((3, 3, 2)), heads.Masked(9), width=16, depth=2)
    opts = training.make_optimizer(net, 'muon', lr=.5, hidden_lr=.25)
    for p in net.parameters():
        p.grad = torch.ones_like(p)
    opts[1].step()
    storage.save(tmp_path / 'x', agent=net, opt=opts)
    state = storage.load(tmp_path / 'x')['opt']
    other = training.make_optimizer(net, 'muon')
    other.load_state_dict(state)
    assert [o.param_groups[0]['lr'] for o in other] == [.25, .5]
    assert torch.equal(other[1].state[net.policy.core.weight]['exp_avg'], opts[1].state[net.policy.core.weight]['exp_avg'])
    with pytest.raises(ValueError):
        other.load_state_dict({'0': state['0']})


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    from boardlaw_amd import heads, networks
    z = lambda *s, dtype=torch.float32: torch.zeros(s, dtype=dtype, device='cuda')
    for bad in (dict(actions=z(2, dtype=torch.int64)), dict(valid=z(3, 5, dtype=torch.bool))):
        with pytest.raises((ValueError, RuntimeError)):
            heads.logprobs(z(3, 4), **bad)
    for bad in (dict(actions=z(3)), dict(valid=z(3, 4, dtype=torch.uint8))):
        with pytest.raises(TypeError):
            heads.logprobs(z(3, 4), **bad)
    with pytest.raises(AssertionError):
        heads.logprobs(z(3, 4), torch.zeros(3, dtype=torch.int64))
    x, y, w = z(3, 4), z(3, 4), z(4)
    for bad in (dict(y=z(3, 5)), dict(y=z(2, 4)), dict(pre=w), dict(y=y, pre=z(5)), dict(y=y, alpha=z(1)), dict(y=y, post=w.half()), dict(y=y, gate=z(3, 3)),
                dict(y=z(3, 8), gate=y), dict(post=w, pre=w), dict(alpha=z(), pre=w), dict(y=y, eps=-1.), dict()):
        if bad == dict(pre=w):
            continue
        with pytest.raises(ValueError):
            networks.norm_residual(x, **bad)
    for bad in (dict(y=y.half(), gate=y), dict(y=y, gate=w.half()), dict(y=y, dtype=torch.half, pre=w)):
        with pytest.raises(TypeError):
            networks.norm_residual(x, **bad)
    with pytest.raises(TypeError):
        networks.norm_residual(x.half(), y, pre=w)


def test_library_refuses_bad_arguments():
    """The C entry points, without a GPU: null pointers, sizes, types, missing workspaces."""
    import ctypes
    from boardlaw_amd import _native
    L, p = _native.lib(), ctypes.c_void_p(16)
    rows = lambda raw=p, dt=0, st=8, R=2, A=8, k=0, act=None, logp=None, ent=p, top=None, tl=None, work=None: L.bl_logprobs(raw, dt, st, None, 0, act, R, A, k, logp, ent, top, tl, None, work, None)
    assert [rows(raw=None), rows(dt=3), rows(R=0), rows(A=0), rows(k=-1), rows(act=p), rows(ent=None), rows(k=2), rows(R=1, A=10000)] == [_native.BL_EINVAL] * 9
    assert rows(k=65, top=p, tl=p) == _native.BL_ETOOBIG and rows(R=1 << 25) == _native.BL_ETOOBIG
    assert L.bl_logprobs_workspace(1, 81, 5) == 0 and L.bl_logprobs_workspace(1, 10000, 5) == 2 * (16 + 40)
    grad = lambda **kw: L.bl_logprobs_grad(*[kw.get(n, d) for n, d in (('raw', p), ('dt', 0), ('st', 8), ('valid', None), ('vs', 0), ('act', None), ('R', 2), ('A', 8), ('k', 0), ('top', None),
                                                                     ('stats', p), ('ent', p), ('gl', None), ('ge', None), ('gt', None), ('d', p), ('s', None))])
    assert [grad(stats=None), grad(ent=None), grad(d=None), grad(gl=p), grad(gt=p, k=2)] == [_native.BL_EINVAL] * 5
    norm = lambda **kw: L.bl_norm_residual(*[kw.get(n, d) for n, d in (('x', p), ('tx', 0), ('xs', 8), ('y', p), ('ty', 0), ('ys', 8), ('al', None), ('post', None), ('gate', None), ('kind', 0),
                                                                     ('gs', 0), ('pre', p), ('eps', 1e-5), ('R', 2), ('W', 8), ('xo', p), ('h', p), ('st', None), ('s', None))])
    assert [norm(x=None), norm(R=0), norm(W=0), norm(eps=-1.), norm(eps=math.nan), norm(kind=1), norm(gate=p), norm(kind=4, gate=p), norm(xo=None), norm(h=None), norm(y=None),
            norm(tx=1, ty=0), norm(ty=3), norm(xs=-1)] == [_native.BL_EINVAL] * 14
    assert norm(W=8193) == _native.BL_ETOOBIG
    arr = (ctypes.c_void_p * 1)(16)
    ortho = lambda **kw: L.bl_orthogonalize(*[kw.get(n, d) for n, d in (('i', arr), ('o', arr), ('c', 1), ('dt', 0), ('m', 8), ('n', 8), ('steps', 5), ('eps', 1e-7), ('work', p), ('s', None))])
    assert [ortho(i=None), ortho(o=None), ortho(c=0), ortho(dt=5), ortho(m=0), ortho(steps=0), ortho(eps=-1.), ortho(work=None), ortho(i=(ctypes.c_void_p * 1)(None))] == [_native.BL_EINVAL] * 9
    assert ortho(m=16385) == _native.BL_ETOOBIG
