"""Flat multi-tensor optimizer kernels (``optimizer.hip``) and sparse row updates."""
from __future__ import annotations

import torch

from . import fn, native, stream_ptr, check, check_device, ptr, record_native, P, I64, I32, F32

MODES = dict(sgd=0, momentum=1, nesterov=2, adagrad=3, adam=4, adamw=5, lamb=6)


def optimizer_flat(mode, p, g, s1=None, s2=None, shadow=None, lr=0.01, l2=0.0, mu=0.9,
                   beta1=0.9, beta2=0.999, beta1t=1.0, beta2t=1.0, eps=1e-7, wd=0.0,
                   gscale=1.0, seg_off=None, seg_off_host=None, norms_ws=None, dyn=None):
    """Update flat fp32 ``p`` in place from flat fp32 ``g``.

    ``seg_off`` (device int64, LAMB only) holds per-tensor offsets.  ``shadow``
    (bf16, same numel) receives the updated weights for mixed precision.
    """
    m = MODES[mode]
    from . import deterministic
    # deterministic LAMB: the per-tensor norms as ordered torch reductions below
    # instead of the fused kernel's cross-block atomics
    if native(p) and not (mode == 'lamb' and deterministic()):
        f = fn('hetu_optimizer_flat', [I32, P, P, P, P, P, I64, F32, F32, F32, F32, F32, F32, F32,
                                       F32, F32, F32, P, I32, P, P, P])
        nseg = (seg_off.numel() - 1) if seg_off is not None else 0
        check(f(m, p.data_ptr(), g.data_ptr(), s1.data_ptr() if s1 is not None else None,
                s2.data_ptr() if s2 is not None else None,
                shadow.data_ptr() if shadow is not None else None, p.numel(), lr, l2, mu, beta1,
                beta2, beta1t, beta2t, eps, wd, gscale,
                seg_off.data_ptr() if seg_off is not None else None, nseg,
                norms_ws.data_ptr() if norms_ws is not None else None,
                dyn.data_ptr() if dyn is not None else None, stream_ptr()), 'optimizer')
        return
    if dyn is not None:
        lr, beta1t, beta2t, gscale = [float(v) for v in dyn.tolist()[:4]]
    from . import cpu_native
    if mode != 'lamb' and cpu_native.active(p, g) and p.is_contiguous() and g.is_contiguous():
        cpu_native.optimizer(mode, p, g, s1, s2, lr, l2, mu, beta1, beta2, beta1t, beta2t, eps, wd, gscale)
        if shadow is not None:
            shadow.copy_(p)
        return
    gr = g * gscale + l2 * p if (gscale != 1.0 or l2) else g
    if mode == 'sgd':
        p.sub_(lr * gr)
    elif mode == 'momentum':
        s1.mul_(mu).sub_(lr * gr)
        p.add_(s1)
    elif mode == 'nesterov':
        t = lr * gr
        s1.sub_(t).mul_(mu)
        p.add_(s1 - t)
    elif mode == 'adagrad':
        s1.add_(gr * gr)
        p.sub_(lr * gr / (torch.sqrt(s1) + eps))
    else:
        s1.mul_(beta1).add_((1 - beta1) * gr)
        s2.mul_(beta2).add_((1 - beta2) * gr * gr)
        u = (s1 / (1 - beta1t)) / (torch.sqrt(s2 / (1 - beta2t)) + eps)
        if mode == 'adam':
            p.sub_(lr * u)
        elif mode == 'adamw':
            p.sub_(lr * (u + wd * p))
        else:  # lamb, per segment
            offs = seg_off_host
            for i in range(len(offs) - 1):
                a, b = offs[i], offs[i + 1]
                pn = torch.linalg.vector_norm(p[a:b])
                un = torch.linalg.vector_norm(u[a:b])
                ratio = (pn / un) if (pn > 0 and un > 0) else torch.tensor(1.0)
                p[a:b].sub_(lr * ratio * (u[a:b] + wd * p[a:b]))
    if shadow is not None:
        shadow.copy_(p)


# ---- AdamW with both moments in 8 bits (adamw8.hip) ---------------------------------------------
_ADAMW8 = [P, P, P, P, P, P, P, I64] + [F32] * 10 + [P, I64, P]
STATE8_BLOCK = 256      # consecutive elements that share the moments' scales


_M64 = (1 << 64) - 1


def _i64(seed):
    """the low 64 bits as a signed launch argument"""
    seed = int(seed) & _M64
    return seed - (1 << 64) if seed >> 63 else seed


# step numbers that fp32 holds one by one: the seeds start again beyond them, for a captured step has
# its number as fp32
STEP_SEEDS = 1 << 24


def step_seed(seed, step):
    """the rounding seed of one step (of step modulo 2^24)"""
    return (int(seed) + int(step) % STEP_SEEDS * 0x9E3779B97F4A7C15) & _M64


def adamw8_state(n, device):
    """(m, v, m_scale, v_scale) of ``n`` weights before their first step: all zero.  ``m`` holds
    float8_e4m3fn, ``v`` float8_e5m2 values; element i stands for value[i] * scale[i // 256]."""
    from .. import native_array as _NA
    nb = -(-int(n) // STATE8_BLOCK)
    return (_NA.zeros(int(n), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn),
            _NA.zeros(int(n), dtype=torch.uint8, device=device).view(torch.float8_e5m2),
            _NA.zeros(nb, dtype=torch.float32, device=device), _NA.zeros(nb, dtype=torch.float32, device=device))


def state8_values(q, scale):
    """the fp32 values that an 8-bit moment stands for"""
    return q.float() * scale.repeat_interleave(STATE8_BLOCK)[:q.numel()]


def state8_from_values(x, which):
    """(8-bit values, block scales) nearest to fp32 ``x``: a moment's form ('s1': the first, 's2':
    the second) made from 32 bits, as when a checkpoint with 32-bit moments is resumed"""
    first = which == 's1'
    x = x.reshape(-1).float()
    nb = -(-x.numel() // STATE8_BLOCK)
    scale = _scale8(x, nb, 7 if first else 14)
    y = x / scale.repeat_interleave(STATE8_BLOCK)[:x.numel()]
    if not first:       # the smallest value above 0 stays above 0
        y = torch.where((x > 0) & (y < 2.0 ** -16), torch.full_like(y, 2.0 ** -16), y)
    return y.to(torch.float8_e4m3fn if first else torch.float8_e5m2), scale


def _round_bits(n, seed, device):
    """adamw8.hip ``round_bits`` of elements 0 .. n - 1"""
    h = (torch.arange(n, device=device) * 0x9E3779B1 + seed) & 0xFFFFFFFF
    h = ((h ^ (h >> 16)) * 0x7FEB352D) & 0xFFFFFFFF
    h = ((h ^ (h >> 15)) * 0x846CA68B) & 0xFFFFFFFF
    return h ^ (h >> 16)


def _encode8(y, r16, mant, bias):
    """adamw8.hip ``encode_m`` / ``encode_v``: codes of y = |x| / scale, whose bits once it is
    multiplied by 2^(bias - 127) are the code's, with the part to be cut off below"""
    cut = 23 - mant
    r = ((r16 << (cut - 16)) | (1 << (cut - 17))).int()
    y = torch.where(torch.isfinite(y), y, torch.zeros_like(y)) * 2.0 ** (bias - 127)
    return (y.view(torch.int32) + r) >> cut


def _scale8(x, nb, top):
    x = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x))
    x = torch.nn.functional.pad(x, (0, nb * STATE8_BLOCK - x.numel())).view(nb, STATE8_BLOCK)
    return (((x.amax(1).view(torch.int32) >> 23) - top).clamp_min(1) << 23).view(torch.float32)


def adamw8(p, g, m, v, m_scale, v_scale, shadow=None, *, lr, beta1=0.9, beta2=0.999, beta1t=0.0, beta2t=0.0,
           eps=1e-7, wd=0.0, gscale=1.0, seed=0, dyn=None):
    """One AdamW step of the flat fp32 weights ``p`` from the flat fp32 gradients ``g``, in place,
    with both moments in 8 bits (``adamw8_state``).

    The update takes the fresh moments in 32 bits; what is stored of them is rounded at random,
    by bits that a hash of ``seed`` (64 bits) and the element's index gives: another seed every
    step.  ``dyn``: fp32 {lr, beta1t, beta2t, gscale, step, 1 - beta1t, 1 - beta2t} on the device
    instead of the arguments, for a captured step; the seed is then moved by ``step`` (modulo
    ``STEP_SEEDS``) as ``step_seed`` moves it.
    ``shadow`` (bf16, the weights' copy) is written too.  A block of 256 shares one scale: where
    several tensors share the buffer, start each at a multiple of 256.  ``eps`` is at least 1e-12."""
    n = p.numel()
    nb = -(-n // STATE8_BLOCK)
    for t, dt, size, what in ((p, torch.float32, n, 'p'), (g, torch.float32, n, 'g'), (m, torch.float8_e4m3fn, n, 'm'),
                              (v, torch.float8_e5m2, n, 'v'), (m_scale, torch.float32, nb, 'm_scale'),
                              (v_scale, torch.float32, nb, 'v_scale'), (shadow, torch.bfloat16, n, 'shadow'),
                              (dyn, torch.float32, 7, 'dyn')):
        if t is None:
            continue
        if t.dtype != dt or t.numel() != size or not t.is_contiguous() or t.device != p.device:
            raise ValueError('adamw8: %s has to be a contiguous %s of %d elements on %s, got %s %s on %s'
                             % (what, dt, size, p.device, t.dtype, tuple(t.shape), t.device))
    if not eps >= 1e-12:
        raise ValueError('adamw8: eps has to be at least 1e-12, got %r' % (eps,))
    if n == 0:
        return
    if native(p):
        check_device(p, 'adamw8')
        f = fn('hetu_adamw8', _ADAMW8)
        check(f(p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(), m_scale.data_ptr(), v_scale.data_ptr(),
                ptr(shadow), n, lr, beta1, beta2, 1.0 - beta1, 1.0 - beta2, 1.0 - beta1t, 1.0 - beta2t, eps,
                wd, gscale, ptr(dyn), _i64(seed), stream_ptr()), 'adamw8')
        record_native('adamw8')
        return
    if dyn is not None:
        lr, _, _, gscale, step, c1, c2 = [float(x) for x in dyn.tolist()]
        seed = step_seed(seed, step)
    else:
        c1, c2 = 1.0 - beta1t, 1.0 - beta2t
    key = int(seed) & _M64
    r = _round_bits(n, (key ^ (key >> 32)) & 0xFFFFFFFF, p.device)
    gr = g * gscale
    m1 = beta1 * state8_values(m, m_scale) + (1 - beta1) * gr
    v1 = beta2 * state8_values(v, v_scale) + (1 - beta2) * gr * gr
    u = (m1 / c1) / (torch.sqrt(v1 / c2) + eps)
    p.sub_(lr * (u + wd * p))
    if shadow is not None:
        shadow.copy_(p)
    m_scale.copy_(_scale8(m1, nb, 7))
    v_scale.copy_(_scale8(v1, nb, 14))
    mc = _encode8(m1.abs() / m_scale.repeat_interleave(STATE8_BLOCK)[:n], r & 0xFFFF, 3, 7)
    mc = torch.where(torch.isfinite(m1), mc, torch.full_like(mc, 0x7F)) | ((m1 < 0).int() << 7)
    vc = _encode8(v1 / v_scale.repeat_interleave(STATE8_BLOCK)[:n], r >> 16, 2, 15)
    vc = torch.where(v1 > 0, vc.clamp_min(1), vc)
    vc = torch.where(torch.isnan(v1), torch.full_like(vc, 0x7F), torch.where(torch.isinf(v1), torch.full_like(vc, 0x7C), vc))
    m.view(torch.uint8).copy_(mc)
    v.view(torch.uint8).copy_(vc)


SPARSE_MODES = dict(sgd=0, momentum=1, nesterov=2, adagrad=3, adam=4, adamw=5)


def sparse_update(mode, table, ids, grads, s1=None, s2=None, lr=0.01, l2=0.0, mu=0.9,
                  beta1=0.9, beta2=0.999, beta1t=1.0, beta2t=1.0, eps=1e-7, wd=0.0):
    """Row-sparse update of ``table`` (fp32 [rows, dim]) at UNIQUE ``ids``."""
    dim = table.shape[-1]
    g = grads.reshape(-1, dim).float().contiguous()
    ids = ids.reshape(-1).long().contiguous()
    if native(table):
        f = fn('hetu_sparse_opt', [I32, P, P, P, P, P, I64, I64, I64, F32, F32, F32, F32, F32,
                                   F32, F32, F32, F32, P])
        check(f(SPARSE_MODES[mode], table.data_ptr(), s1.data_ptr() if s1 is not None else None,
                s2.data_ptr() if s2 is not None else None, ids.data_ptr(), g.data_ptr(),
                ids.numel(), dim, table.shape[0], lr, l2, mu, beta1, beta2, beta1t, beta2t, eps,
                wd, stream_ptr()), 'sparse_opt')
        return
    # ids < 0 mark rows the dense de-duplication left untouched (optimizer.py);
    # the native kernel skips them, the torch path must too (table[-1] is a real row)
    keep = ids >= 0
    if not bool(keep.all()):
        ids, g = ids[keep], g[keep]
    p = table[ids]
    gr = g + l2 * p if l2 else g
    if mode == 'sgd':
        p = p - lr * gr
    elif mode == 'momentum':
        v = mu * s1[ids] - lr * gr
        s1[ids] = v
        p = p + v
    elif mode == 'nesterov':
        t = lr * gr
        v = mu * (s1[ids] - t)
        s1[ids] = v
        p = p + v - t
    elif mode == 'adagrad':
        a = s1[ids] + gr * gr
        s1[ids] = a
        p = p - lr * gr / (torch.sqrt(a) + eps)
    else:
        m = beta1 * s1[ids] + (1 - beta1) * gr
        v = beta2 * s2[ids] + (1 - beta2) * gr * gr
        s1[ids] = m
        s2[ids] = v
        u = (m / (1 - beta1t)) / (torch.sqrt(v / (1 - beta2t)) + eps)
        p = p - lr * u if mode == 'adam' else p - lr * (u + wd * p)
    table[ids] = p
