"""Observation intakes and policy/value heads for the leaf-evaluation network (PyTorch-ROCm; the GEMMs are the only
MFMA work on the path).  Mirrors the parts of boardlaw/heads.py the Hex path reaches -- space tuples
(heads.py:7-11), the flattening Linear intake (heads.py:41-52), the masked log-softmax policy head (heads.py:92-104),
the seat-scattered tanh value head (heads.py:128-142) -- with the same parameter names, so reference checkpoints load."""
from collections import namedtuple

import numpy as np
import torch
from torch import nn
from torch.autograd.function import once_differentiable
from torch.nn import functional as F

from . import _native, arrdict

Empty = namedtuple('Empty', ())
Discrete = namedtuple('Discrete', ('dim',))
Masked = namedtuple('Masked', ('dim',))
Vector = namedtuple('Vector', ('dim',))
Tensor = namedtuple('Tensor', ('dim',))


class _FlatLinear(nn.Linear):
    """Linear over the trailing `event_ndim` dims, for inputs shaped (B, *event) or (T, B, *event)."""

    def __init__(self, event_shape, width):
        self._event_ndim = len(event_shape)
        super().__init__(int(np.prod(event_shape)), width)

    def forward(self, obs, *args, **kwargs):
        lead = obs.shape[:obs.ndim - self._event_ndim]
        return super().forward(obs.reshape(*lead, -1))


class TensorIntake(_FlatLinear):
    def __init__(self, space, width):
        super().__init__(tuple(space.dim), width)


class VectorIntake(_FlatLinear):
    def __init__(self, space, width):
        super().__init__(tuple(space.dim), width)


def intake(space, width):
    kinds = {'Tensor': TensorIntake, 'Vector': VectorIntake}
    name = type(space).__name__
    if name not in kinds:
        raise ValueError(f"Can't handle {space}")
    return kinds[name](space, width)


def _logprobs(raw, actions, valid, k, want_stats):
    R, A = raw.shape
    dev = raw.device
    new = lambda *shape, dtype=torch.float32: torch.empty(shape, dtype=dtype, device=dev)
    logp = new(R) if actions is not None else None
    entropy = new(R)
    top, top_logp = (new(R, k, dtype=torch.int64), new(R, k)) if k else (None, None)
    stats = new(R, 2) if want_stats else None
    if R:
        L = _native.lib()
        size = L.bl_logprobs_workspace(R, A, k)
        work = new(size, dtype=torch.uint8) if size else None
        p = lambda t: None if t is None else t.data_ptr()
        with _native.on(dev):
            _native.check(L.bl_logprobs(raw.data_ptr(), _native.DTYPES[raw.dtype], raw.stride(0), p(valid), 0 if valid is None else valid.stride(0),
                                        p(actions), R, A, k, p(logp), entropy.data_ptr(), p(top), p(top_logp), p(stats), p(work), _native.stream(dev)))
    return logp, entropy, top, top_logp, stats


class _LogProbs(torch.autograd.Function):

    @staticmethod
    def forward(ctx, raw, actions, valid, k):
        logp, entropy, top, top_logp, stats = _logprobs(raw, actions, valid, k, True)
        ctx.k = k
        ctx.save_for_backward(raw, actions, valid, top, stats, entropy)
        ctx.set_materialize_grads(False)
        if top is not None:
            ctx.mark_non_differentiable(top)
        return logp, entropy, top, top_logp

    @staticmethod
    @once_differentiable
    def backward(ctx, g_logp, g_entropy, g_top, g_top_logp):
        raw, actions, valid, top, stats, entropy = ctx.saved_tensors
        R, A = raw.shape
        d = torch.empty((R, A), dtype=raw.dtype, device=raw.device)
        if R:
            gs = [None if g is None else g.float().contiguous() for g in (g_logp, g_entropy, g_top_logp)]
            p = lambda t: None if t is None else t.data_ptr()
            with _native.on(raw.device):
                _native.check(_native.lib().bl_logprobs_grad(
                    raw.data_ptr(), _native.DTYPES[raw.dtype], raw.stride(0), p(valid), 0 if valid is None else valid.stride(0), p(actions), R, A, ctx.k,
                    p(top), stats.data_ptr(), entropy.data_ptr(), p(gs[0]), p(gs[1]), p(gs[2]), d.data_ptr(), _native.stream(raw.device)))
        return d, None, None, None


def logprobs(raw, actions=None, valid=None, k=0):
    """Log probabilities of given moves, entropy and the best alternatives of policy rows, in one pass over the logits:

        raw      (..., A) unnormalised logits, f32 / f16 / bf16
        actions  (...) whole numbers: the given moves; -1 where a row has none (padding)
        valid    (..., A) bool, or what broadcasts to it: invalid moves have probability 0 whatever `raw` holds there.  A logit of -inf is an invalid move.
        k        how many alternatives, up to 64

    -> arrdict of f32 `logp` (...) (with actions), `entropy` (...), `top` (..., k) int64 and `top_logp` (..., k) (with k).  The alternatives come
    in descending order, equal ones by index; where fewer than k moves are valid the rest is -1 and -inf.  An invalid given move
    has logp -inf, a missing one (-1) 0, one beyond the row NaN.  A row with no valid move has entropy 0.  Differentiable (once) in `raw` through
    logp, entropy and top_logp; an invalid move's gradient is 0.  On the GPU only (bl_logprobs)."""
    if raw.dtype not in _native.DTYPES:
        raise TypeError(f'raw must be float32, float16 or bfloat16, got {raw.dtype}')
    if raw.ndim < 1 or raw.shape[-1] < 1:
        raise ValueError(f'raw must be (..., A) with at least one move, got {tuple(raw.shape)}')
    if not 0 <= k <= _native.TOP_MAX:
        raise ValueError(f'k must be in 0 .. {_native.TOP_MAX}, got {k}')
    _native.require_device(*(t for t in (raw, actions, valid) if t is not None))
    lead, A = raw.shape[:-1], raw.shape[-1]
    flat = _native.rows_of(raw, A)
    if actions is not None:
        if actions.shape != lead:
            raise ValueError(f'actions must be {tuple(lead)}, got {tuple(actions.shape)}')
        if actions.is_floating_point() or actions.is_complex() or actions.dtype == torch.bool:
            raise TypeError(f'actions must be whole numbers, got {actions.dtype}')
        actions = actions.long().reshape(-1).contiguous()
    if valid is not None:
        if valid.dtype != torch.bool:
            raise TypeError(f'valid must be bool, got {valid.dtype}')
        valid = _native.rows_of(valid.expand(raw.shape), A)
    if torch.is_grad_enabled() and raw.requires_grad:
        logp, entropy, top, top_logp = _LogProbs.apply(flat, actions, valid, k)
    else:
        logp, entropy, top, top_logp, _ = _logprobs(flat.detach(), actions, valid, k, False)
    out = arrdict.arrdict()
    if logp is not None:
        out['logp'] = logp.view(lead)
    out['entropy'] = entropy.view(lead)
    if k:
        out['top'], out['top_logp'] = top.view(*lead, k), top_logp.view(*lead, k)
    return out


class _PolicyHead(nn.Module):
    def __init__(self, space, width):
        super().__init__()
        self.shape = (space.dim,) if np.isscalar(space.dim) else tuple(space.dim)
        self.core = nn.Linear(width, int(np.prod(self.shape)))

    def raw(self, x):
        return self.core(x).reshape(*x.shape[:-1], *self.shape)

    def sample(self, logits, test=False):
        return logits.argmax(-1) if test else torch.distributions.Categorical(logits=logits).sample()

    def evaluate(self, x, valid=None, actions=None, k=0):
        """logprobs() of this head's outputs for the neck `x`: what forward() normalises, without the (B, A) result."""
        y, lead = self.core(x), x.shape[:-1]
        return logprobs(y, actions, None if valid is None else valid.reshape(*lead, -1), k)


class DiscreteOutput(_PolicyHead):
    def forward(self, x, *args, **kwargs):
        return F.log_softmax(self.raw(x), -1)


class MaskedOutput(_PolicyHead):
    """Invalid actions get logit -inf, hence probability exactly 0 in the search (the kernels see no mask)."""

    def forward(self, x, valid, *args, **kwargs):
        y = self.raw(x)
        return F.log_softmax(y.masked_fill(~valid, -np.inf), -1)


def output(space, width):
    kinds = {'Discrete': DiscreteOutput, 'Masked': MaskedOutput}
    name = type(space).__name__
    if name not in kinds:
        raise ValueError(f"Can't handle {space}")
    return kinds[name](space, width)


def scatter_values(v, seats):
    """Puts +v at the mover's seat and -v at the other one: (B,) -> (B,2).  heads.py:122-126"""
    idx = torch.stack([seats, 1 - seats], -1).long()
    return torch.full_like(torch.stack([v, -v], -1), np.nan).scatter(-1, idx, torch.stack([v, -v], -1))


class ValueOutput(nn.Module):
    def __init__(self, width):
        super().__init__()
        self.core = nn.Linear(width, 1)

    def forward(self, x, valid, seats, *args, **kwargs):
        return scatter_values(torch.tanh(self.core(x).squeeze(-1)), seats)
