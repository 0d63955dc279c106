"""The learner's optimiser for hidden weights: momentum updates orthogonalised by Newton-Schulz products before they are applied.  The
reference trains with Adam alone (boardlaw/main.py:153); here `training.run(optimizer='muon')` gives the residual blocks' weights
to Muon and everything else to Adam."""
import torch

from . import _native, networks


def orthogonalize(matrices, steps=5, eps=1e-7):
    """The Newton-Schulz iteration X = aX + (bA + cA^2)X, A = XX^T, from X = G / (|G| + eps): the matrix with G's singular vectors and singular
    values near 1 (0.7 .. 1.2 after five steps; those under about 1e-3 of |G| have not got there yet).

        matrices  a tensor (..., m, n), or a list of matrices (m, n) of any shapes: f32, f16 or bf16, sides up to 16384

    -> the same structure, types and shapes; as exact as f32 products whatever the type (22-bit operands and f32 sums; f64 for a shorter side of up to
    32, or up to 64 beside more than 128, and up to 6 steps).  Matrices of one shape and type are taken through it together.  Not differentiable.  On the GPU only (bl_orthogonalize)."""
    if not isinstance(matrices, torch.Tensor):
        return _native.ops().orthogonalize(matrices, steps, eps)
    if matrices.ndim < 2:
        raise ValueError(f'a matrix or a batch of them is wanted, got {tuple(matrices.shape)}')
    if matrices.ndim == 2:
        return _native.ops().orthogonalize([matrices], steps, eps)[0]
    flat = matrices.detach().reshape(matrices.shape[:-2].numel(), *matrices.shape[-2:])
    if flat.shape[0] == 0:
        _native.require_device(matrices)
        return torch.empty_like(matrices)
    return torch.stack(_native.ops().orthogonalize(list(flat.unbind(0)), steps, eps)).view(matrices.shape)


class Muon(torch.optim.Optimizer):
    """Momentum SGD whose update of every weight matrix is orthogonalised: m = momentum m + g, u = g + momentum m (nesterov) or m,
    W = (1 - lr weight_decay) W - lr sqrt(max(1, rows / cols)) orthogonalize(u).  For the two-dimensional weights of hidden layers.  m is held in the
    weights' type, which is f32 in this package's networks."""

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0., steps=5):
        if not lr >= 0 or not 0 <= momentum < 1 or not weight_decay >= 0:
            raise ValueError(f'lr and weight_decay must not be negative, momentum in [0, 1): got {lr}, {weight_decay}, {momentum}')
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps))
        for group in self.param_groups:
            for p in group['params']:
                if p.ndim != 2:
                    raise ValueError(f'Muon is for matrices, got a parameter of shape {tuple(p.shape)}')

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            params = [p for p in group['params'] if p.grad is not None]
            if not params:
                continue
            grads = [p.grad for p in params]
            moments = []
            for p in params:
                state = self.state[p]
                if 'momentum' not in state:
                    state['momentum'] = torch.zeros_like(p, memory_format=torch.preserve_format)
                moments.append(state['momentum'])
            torch._foreach_mul_(moments, group['momentum'])
            torch._foreach_add_(moments, grads)
            updates = torch._foreach_add(grads, moments, alpha=group['momentum']) if group['nesterov'] else moments
            updates = orthogonalize(updates, steps=group['steps'])
            if group['weight_decay']:
                torch._foreach_mul_(params, 1 - group['lr'] * group['weight_decay'])
            scales = {}
            for p, u in zip(params, updates):
                ps, us = scales.setdefault(max(1., p.shape[0] / p.shape[1]) ** .5, ([], []))
                ps.append(p); us.append(u)
            for scale, (ps, us) in scales.items():
                torch._foreach_add_(ps, us, alpha=-group['lr'] * scale)
        return loss


class Several(tuple):
    """Optimisers that share a network's parameters out among them, as training.optimize takes them: saved and loaded as one (storage.save(opt=...)), and
    one to a GradScaler, which looks through all parameter groups and steps all of them or none."""

    @property
    def param_groups(self):
        return [group for o in self for group in o.param_groups]

    def zero_grad(self, set_to_none=True):
        for o in self:
            o.zero_grad(set_to_none)

    def step(self):
        for o in self:
            o.step()

    def state_dict(self):
        return {str(i): o.state_dict() for i, o in enumerate(self)}

    def load_state_dict(self, state):
        if len(state) != len(self):
            raise ValueError(f'a state of {len(state)} optimisers for {len(self)}')
        for i, o in enumerate(self):
            o.load_state_dict(state[str(i)])


def split(network):
    """A network's parameters as (hidden weight matrices, the rest): the residual blocks' weights are Muon's, biases, gains, the intake
    and the heads Adam's."""
    hidden = [m.weight for m in network.modules() if isinstance(m, (networks.ReZeroResidual, networks.GatedResidual))]
    ids = {id(p) for p in hidden}
    return hidden, [p for p in network.parameters() if id(p) not in ids]
