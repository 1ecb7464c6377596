"""Log probabilities of given tokens with entropy and most probable tokens, and their gradient
(``logprob.hip``)."""
from __future__ import annotations

import math

import torch
from .. import native_array as _NA

from . import fn, native, stream_ptr, is_bf16, check, check_device, ptr, supported_float, record_native, P, I64, I32

MAX_TOP = 64
_FWD = [P, I64, P, I64, I32, I32, I64, P, P, I32, P]
_BWD = [P, I64, P, I64, I32, I32, I64, P, P, P, P, I32, P]


class TokenLogProb(object):
    """Result of ``token_logprob`` for logits [..., V]: ``logp`` [...], ``entropy`` [...] and
    ``top_logp`` [..., top], all columns of ``out`` (fp32 [..., 2 + top]); ``top_ids`` [..., top]
    (int64); ``stats`` [..., 2], each row's maximum and base-2 log of its sum, for the backward
    pass.  The fp32 parts are views of one buffer [..., 4 + top]."""
    __slots__ = ('buffer', 'ids')

    def __init__(self, buffer, ids):
        self.buffer, self.ids = buffer, ids

    @property
    def top_ids(self):
        if self.ids is None:           # no alternatives
            return self.buffer.new_empty(self.buffer.shape[:-1] + (0,), dtype=torch.int64)
        return self.ids

    @property
    def top(self):
        return self.buffer.shape[-1] - 4

    @property
    def out(self):
        return self.buffer[..., :-2]

    @property
    def stats(self):
        return self.buffer[..., -2:]

    @property
    def logp(self):
        return self.buffer[..., 0]

    @property
    def entropy(self):
        return self.buffer[..., 1]

    @property
    def top_logp(self):
        return self.buffer[..., 2:-2]


def _operands(name, logits, ids, top):
    if not isinstance(logits, torch.Tensor) or logits.dim() < 1 or not supported_float(logits):
        raise ValueError('%s: logits have to be an fp32 or bf16 tensor of at least one dimension' % name)
    V = logits.shape[-1]
    if not 1 <= V < 2 ** 31 - 64:
        raise ValueError('%s: a row has 1 to 2^31 - 65 logits, got %d' % (name, V))
    if not 0 <= top <= min(MAX_TOP, V):
        raise ValueError('%s: top is 0 to min(%d, %d), got %d' % (name, MAX_TOP, V, top))
    two = logits.dim() == 2
    lead = (logits.shape[0],) if two else tuple(logits.shape[:-1])
    R = lead[0] if two else math.prod(lead)
    if ids.numel() != R or ids.is_floating_point() and ids.dtype not in (torch.float32, torch.float64):
        raise ValueError('%s: one token id a row: %d rows, ids %s %s' % (name, R, tuple(ids.shape), ids.dtype))
    if ids.device != logits.device:
        raise ValueError('%s: logits on %s, ids on %s' % (name, logits.device, ids.device))
    x = logits if two else logits.reshape(R, V)
    if V > 1 and x.stride(1) != 1:
        x = x.contiguous()
    if ids.dim() != 1:
        ids = ids.reshape(R)
    if ids.dtype != torch.int64:
        ids = ids.long()
    return x, ids.contiguous(), lead, R, V


def _stride(x):
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def token_logprob(logits, ids, top=0, ignored_index=-1):
    """For each row of ``logits`` [..., V] (fp32 or bf16; rows may be strided): the log probability
    of token ``ids`` [...], the row's entropy (both in nats) and its ``top`` (0 to 64) largest log
    probabilities with their tokens, in falling order, equal ones by rising token.

    A row whose id is ``ignored_index`` or outside [0, V) is not read: logp, entropy and top_logp
    are 0, top_ids -1.  A row with nothing above -inf has logp and top_logp -inf and entropy 0.
    A NaN or +inf makes its row NaN."""
    x, ids, lead, R, V = _operands('token_logprob', logits, ids, top)
    r = TokenLogProb(_NA.empty(lead + (4 + top,), dtype=torch.float32, device=x.device),
                     _NA.empty(lead + (top,), dtype=torch.int64, device=x.device) if top else None)
    if R == 0:
        return r
    if native(x):
        check_device(x, 'token_logprob')
        f = fn('hetu_token_logprob', _FWD)
        check(f(x.data_ptr(), _stride(x), ids.data_ptr(), R, V, top, ignored_index, r.buffer.data_ptr(), ptr(r.ids),
                is_bf16(x), stream_ptr()), 'token_logprob')
        record_native('token_logprob')
        return r
    xf = x.float()
    valid = (ids >= 0) & (ids < V) & (ids != ignored_index)
    m = xf.amax(1, keepdim=True)
    z = xf - torch.where(m == -math.inf, torch.zeros_like(m), m)
    e = torch.exp(z)
    s = e.sum(1, keepdim=True)
    logs = torch.log(s)
    empty = (s == 0)[:, 0]
    h = logs[:, 0] - (e * z.clamp_min(-200.0)).sum(1) / s[:, 0]
    res = torch.cat([z.gather(1, torch.where(valid, ids, torch.zeros_like(ids))[:, None]) - logs, h[:, None]], 1)
    if top:
        order = torch.where(torch.isnan(xf), torch.full_like(xf, -math.inf), xf)
        idx = torch.sort(order, dim=1, descending=True, stable=True)[1][:, :top]
        res = torch.cat([res, z.gather(1, idx) - logs], 1)
        r.top_ids.copy_(torch.where(valid[:, None], idx, torch.full_like(idx, -1)).reshape(r.top_ids.shape))
    res[empty] = -math.inf
    res[empty, 1] = 0.0
    res[~valid] = 0.0
    st = torch.cat([m, torch.log2(s)], 1)
    st[~valid] = 0.0
    r.buffer.copy_(torch.cat([res, st], 1).reshape(r.buffer.shape))
    return r


def token_logprob_backward(logits, ids, fwd, grad, ignored_index=-1):
    """d logits (contiguous, of the logits' type) from ``grad`` [..., 2 + top], the gradient of
    ``fwd.out``: of logp, of the entropy and of each of ``fwd``'s alternatives.  ``fwd`` is what
    ``token_logprob`` gave for the same logits, ids and ignored_index."""
    top = fwd.top
    x, ids, lead, R, V = _operands('token_logprob_backward', logits, ids, top)
    if tuple(fwd.buffer.shape) != lead + (4 + top,) or grad.numel() != R * (2 + top) or grad.device != x.device:
        raise ValueError('token_logprob_backward: logits %s, forward of %s, gradient %s'
                         % (tuple(logits.shape), tuple(fwd.buffer.shape[:-1]), tuple(grad.shape)))
    for t, shape, dt in ((fwd.buffer, lead + (4 + top,), torch.float32), (fwd.ids, lead + (top,), torch.int64)):
        if t is None and not top:
            continue
        if t is None or tuple(t.shape) != shape or t.dtype != dt or t.device != x.device or not t.is_contiguous():
            raise ValueError('token_logprob_backward: the forward result has to be whole and on %s: %s %s expected, got %s'
                             % (x.device, dt, shape, t if t is None else (t.dtype, tuple(t.shape), t.device)))
    if grad.dtype != torch.float32 or not grad.is_contiguous():
        from .moe import _dc
        grad = _dc(grad, torch.float32)
    dx = _NA.empty(lead + (V,), dtype=x.dtype, device=x.device)
    if R == 0:
        return dx
    if native(x):
        check_device(x, 'token_logprob_backward')
        f = fn('hetu_token_logprob_bwd', _BWD)
        check(f(x.data_ptr(), _stride(x), ids.data_ptr(), R, V, top, ignored_index, fwd.buffer.data_ptr(),
                ptr(fwd.ids), grad.data_ptr(), dx.data_ptr(), is_bf16(x), stream_ptr()), 'token_logprob_bwd')
        record_native('token_logprob_bwd')
        return dx
    g, o = grad.reshape(R, 2 + top), fwd.out.reshape(R, 2 + top)
    m, log2s = fwd.stats.reshape(R, 2)[:, :1], fwd.stats.reshape(R, 2)[:, 1:]
    valid = ((ids >= 0) & (ids < V) & (ids != ignored_index))[:, None]
    dead = ~valid | ((m == -math.inf) & (log2s == -math.inf))
    logq = x.float() - torch.where(m == -math.inf, torch.zeros_like(m), m) - log2s * math.log(2.0)
    d = -torch.exp(logq) * (g[:, :1] + g[:, 2:].sum(1, keepdim=True) + g[:, 1:2] * (logq.clamp_min(-200.0) + o[:, 1:2]))
    d.scatter_add_(1, torch.where(valid, ids[:, None], torch.zeros_like(ids[:, None])), g[:, :1])
    if top:
        d.scatter_add_(1, fwd.top_ids.reshape(R, top).clamp_min(0), g[:, 2:])
    dx.copy_(torch.where(dead, torch.zeros_like(d), d).reshape(dx.shape))
    return dx
