"""Balance loss of a router with per-expert counts: values and gradients against the definition in
64 bits, on the CPU form and the HIP kernels."""
import numpy as np
import pytest
import torch

import hetu_61a7_amd as ht
from hetu_61a7_amd.kernels import moe as K

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]
U = 2.0 ** -24


def _definition(x, idx, valid, g):
    """(loss, counts, d logits) in 64 bits"""
    T, E = x.shape
    on = torch.ones(T, dtype=torch.bool, device=x.device) if valid is None else valid != 0
    q = torch.softmax(x.double(), 1)
    c = idx[on].reshape(-1)
    counts = torch.bincount(c[(c >= 0) & (c < E)], minlength=E)
    n = int(on.sum())
    d = torch.zeros_like(q)
    if n == 0:
        return torch.zeros(1, dtype=torch.float64, device=x.device), counts, d, q, counts.double()
    w = E * counts.double() / n ** 2
    d[on] = g.double() * q[on] * (w - (q[on] @ w)[:, None])
    return (w * q[on].sum(0)).sum().reshape(1), counts, d, q, w


def _case(T, E, k, dt, mask, seed, device):
    g = torch.Generator().manual_seed(seed)
    x = (2.0 * torch.randn(T, E, generator=g) + torch.randn(1, E, generator=g)).to(dt)
    idx = torch.topk(x.float(), k, dim=1)[1]
    if k > 1:
        idx[::7, k - 1] = -1                          # choices not made
    valid = None
    if mask is not None:
        valid = (torch.rand(T, generator=g) < {'most': 0.8, 'none': 0.0, 'one': 0.0}[mask])
        if mask == 'one':
            valid[T // 2] = True
    return x.to(device), idx.to(device), None if valid is None else valid.to(device), torch.rand(1, generator=g).to(device) + 0.5


class _Values(object):
    def __init__(self, loss, counts):
        self.loss, self.counts = loss, counts


def _check(x, idx, valid, g, r, d):
    """p has the roundings of its exponent (at most |x - max| log2 e + 2), of the sum over E (a lane's
    16 terms at most, then joins) and of the quotient; sums over tokens add a lane's share one after
    another: at most T / 512 + 64 terms"""
    T, E = x.shape
    loss, counts, grad, q, w = _definition(x, idx, valid, g)
    assert torch.equal(r.counts, counts)
    span = float((x.double().amax(1, keepdim=True) - x.double()).max()) if T else 0.0
    p = U * (2 * span + 40)
    assert abs(float(r.loss) - float(loss)) <= (p + U * (T / 512 + 64)) * float(loss)
    big = float(w.max()) if E else 0.0
    tol = g.double() * q * (2 * p + U * (E + 16)) * big + 2.0 ** -126
    if d.dtype == torch.bfloat16:
        tol = tol * 1.01 + 2.0 ** -8 * grad.abs()
    assert d.dtype == x.dtype and d.is_contiguous()
    assert bool(((d.double() - grad).abs() <= tol).all())
    if valid is not None:
        assert not d[valid == 0].any()


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dt', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('mask', [None, 'most', 'one', 'none'])
@pytest.mark.parametrize('T,E,k', [(1, 1, 1), (1, 8, 2), (3, 2, 2), (96, 8, 2), (1000, 16, 2), (515, 24, 3), (257, 60, 4),
                                   (100, 161, 6), (33, 256, 8), (77, 512, 8), (20, 513, 1), (9, 1000, 20), (5, 1024, 1),
                                   (40000, 4, 1)])
def test_values_and_gradient(T, E, k, mask, dt, device):
    x, idx, valid, g = _case(T, E, k, dt, mask, 100 * T + E, device)
    r = K.balance_loss(x, idx, E, valid)
    _check(x, idx, valid, g, r, K.balance_loss_backward(x, r, g, valid))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dt', [torch.float32, torch.bfloat16])
def test_strided_logits_and_kinds_of_masks(dt, device):
    for off, E, pitch in ((0, 16, 24), (1, 16, 17), (3, 7, 30), (8, 8, 16)):
        wide, idx, valid, g = _case(300, pitch + off, 2, dt, 'most', E, device)
        x, idx = wide[:, off:off + E], idx.clamp_max(E - 1)
        r = K.balance_loss(x, idx, E, valid)
        d = K.balance_loss_backward(x, r, g, valid)
        _check(x, idx, valid, g, r, d)
        for kind in (torch.uint8, torch.int8, torch.float32, torch.bfloat16, torch.int64, torch.int32):
            v = valid.to(kind) * (3 if kind != torch.bool else 1)
            r2 = K.balance_loss(x, idx, E, v)
            assert torch.equal(r.loss, r2.loss) and torch.equal(r.counts, r2.counts)
            assert torch.equal(d, K.balance_loss_backward(x, r2, g, v))
        every = torch.zeros(600, dtype=torch.bool, device=device)
        every[::2] = valid
        assert torch.equal(K.balance_loss(x, idx, E, every[::2]).loss, r.loss)
        assert torch.equal(K.balance_loss(x, idx.int(), E, valid).loss, r.loss)
        assert torch.equal(K.balance_loss(x, idx.t().contiguous().t(), E, valid).loss, r.loss)
    x, idx, valid, g = _case(40, 40, 2, dt, None, 5, device)
    r = K.balance_loss(x.t(), idx, 40)                # the experts are the strided dimension
    _check(x.t(), idx, None, g, r, K.balance_loss_backward(x.t(), r, g))


@pytest.mark.parametrize('device', DEVICES)
def test_tokens_that_are_not_valid_reach_nothing(device):
    x, idx, valid, g = _case(200, 12, 2, torch.float32, 'most', 1, device)
    r = K.balance_loss(x, idx, 12, valid)
    d = K.balance_loss_backward(x, r, g, valid)
    y, j = x.clone(), idx.clone()
    y[~valid] = float('nan')
    j[~valid] = 2 ** 40
    r2 = K.balance_loss(y, j, 12, valid)
    assert torch.equal(r.loss, r2.loss) and torch.equal(r.counts, r2.counts)
    assert torch.equal(d, K.balance_loss_backward(y, r2, g, valid))


@pytest.mark.parametrize('device', DEVICES)
def test_masked_experts_and_no_tokens(device):
    """an expert at -inf or the lowest value has probability 0 and no gradient"""
    x, idx, _, g = _case(50, 9, 2, torch.float32, None, 2, device)
    for low in (-float('inf'), torch.finfo(torch.float32).min):
        y = x.clone()
        y[:, 4] = low
        j = torch.where(idx == 4, torch.zeros_like(idx), idx)
        r = K.balance_loss(y, j, 9)
        d = K.balance_loss_backward(y, r, g)
        assert not d[:, 4].any()
        loss, counts, grad, q, w = _definition(y, j, None, g)
        assert abs(float(r.loss) - float(loss)) <= 200 * U * float(loss)
        assert bool(((d.double() - grad).abs() <= 200 * U * g.double() * w.max()).all())
    r = K.balance_loss(x[:0], idx[:0], 9)
    assert float(r.loss) == 0 and not r.counts.any()
    assert K.balance_loss_backward(x[:0], r, g).shape == (0, 9)


@pytest.mark.parametrize('device', DEVICES)
def test_gradient_against_differences(device):
    x, idx, valid, g = _case(6, 5, 2, torch.float32, 'most', 3, device)
    r = K.balance_loss(x, idx, 5, valid)
    d = K.balance_loss_backward(x, r, g, valid)
    h = 1e-5
    for i in range(6):
        for j in range(5):
            a, b = x.double().clone(), x.double().clone()
            a[i, j] += h
            b[i, j] -= h
            diff = float(g) * float(_definition(a, idx, valid, g)[0] - _definition(b, idx, valid, g)[0]) / (2 * h)
            assert abs(diff - float(d[i, j])) < 1e-6


def test_refusals():
    x, idx, valid, g = _case(10, 8, 2, torch.float32, 'most', 4, 'cpu')
    for a in ((x.double(), idx, 8), (x[0], idx, 8), (x, idx, 7), (x, idx[:9], 8), (torch.zeros(2, 1025), idx[:2], 1025),
              (x, idx[:, :0], 8), (x, idx, 8, valid[:9]), (x, idx, 8, valid.double())):
        with pytest.raises(ValueError):
            K.balance_loss(*a)
    r = K.balance_loss(x, idx, 8)
    for a in ((x[:, :7], r, g), (x, r, torch.zeros(2)), (x, r, g, valid[:5])):
        with pytest.raises(ValueError):
            K.balance_loss_backward(*a)


@pytest.mark.gpu
def test_same_call_gives_the_same_bits():
    x, idx, valid, g = _case(100003, 60, 4, torch.bfloat16, 'most', 6, 'cuda')
    a = K.balance_loss(x, idx, 60, valid)
    for _ in range(4):
        b = K.balance_loss(x, idx, 60, valid)
        assert torch.equal(a.loss, b.loss) and torch.equal(a.counts, b.counts) and torch.equal(a.weight, b.weight)


# ---- as graph operators ------------------------------------------------------------------------
@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('graph', [False, True])
def test_op(device, graph):
    if graph and device == 'cpu':
        pytest.skip('no captured steps on the CPU')
    x, idx, valid, g = _case(130, 12, 2, torch.float32, 'most', 8, 'cpu')
    X = ht.Variable(name='x', value=x.numpy())
    I, V = ht.Variable(name='i', trainable=False), ht.Variable(name='v', trainable=False)
    loss, counts = ht.balance_loss_op(X, I, 12, V)
    (gx,) = ht.gradients(loss, [X])
    ex = ht.Executor({'train': [loss, counts, gx]}, ctx=ht.cpu(0) if device == 'cpu' else ht.gpu(0), use_hipgraph=graph)
    for _ in range(6 if graph else 1):
        l, c, d = ex.run('train', feed_dict={I: idx.numpy(), V: valid.numpy().astype(np.float32)},
                         convert_to_numpy_ret_vals=True)
        _check(x, idx, valid, torch.ones(1), _Values(torch.from_numpy(l), torch.from_numpy(c)), torch.from_numpy(d))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('fused', [False, True])
def test_gate_with_a_token_mask(device, fused):
    """TopKGate(x, token_mask): the same routing, the balance loss of the tokens that are not padding;
    a mask of ones is the loss without a mask"""
    T, d, E = 24, 8, 4
    rng = np.random.RandomState(0)
    xv = rng.randn(T, d).astype(np.float32)
    out = []
    for mask in (None, np.ones(T, np.float32), (np.arange(T) < 15).astype(np.float32)):
        X, M = ht.Variable(name='x', trainable=False), ht.Variable(name='m', trainable=False)
        gate = ht.layers.TopKGate(d, T, E, k=2, fused=fused, initializer=lambda shape, name: ht.Variable(
            name=name, value=np.random.RandomState(1).randn(*shape).astype(np.float32)))
        l_aux, idx, loc, w, cap = gate(X) if mask is None else gate(X, M)
        ex = ht.Executor({'train': [l_aux] + idx + w}, ctx=ht.cpu(0) if device == 'cpu' else ht.gpu(0))
        r = ex.run('train', feed_dict={X: xv} if mask is None else {X: xv, M: mask}, convert_to_numpy_ret_vals=True)
        out.append([np.asarray(v) for v in r])
    for a, b, c in zip(*[o[1:] for o in out]):
        np.testing.assert_array_equal(a, b)
        np.testing.assert_array_equal(a, c)
    np.testing.assert_allclose(out[0][0].reshape(-1), out[1][0], rtol=100 * U)
    logits = xv @ np.random.RandomState(1).randn(d, E).astype(np.float32)
    q = np.exp(logits - logits.max(1, keepdims=True)).astype(np.float64)
    q /= q.sum(1, keepdims=True)
    top = np.argsort(-logits, 1, kind='stable')[:15, :2]
    want = E * (np.bincount(top.reshape(-1), minlength=E) / 15 * q[:15].mean(0)).sum()
    assert abs(float(out[2][0].reshape(-1)[0]) - want) < 1e-5 * want


def test_mask_is_refused_by_other_gates():
    layer = ht.layers.MoELayer(ht.layers.KTop1Gate(8, 24, 4, k=2), [ht.layers.Expert(8, 8)], 24, 8)
    with pytest.raises(ValueError):
        layer(ht.Variable(name='x'), ht.Variable(name='m'))


@pytest.mark.gpu
def test_fed_choices_keep_their_experts_under_mixed_precision():
    """choices fed as fp32 are labels: no cast to bf16, which holds whole numbers up to 256 alone"""
    T, E = 1200, 600
    rng = np.random.RandomState(2)
    xv, iv = rng.randn(T, E).astype(np.float32), rng.randint(0, E, (T, 2))
    X, I, V = ht.Variable(name='x', value=xv), ht.Variable(name='i', trainable=False), ht.Variable(name='v', trainable=False)
    loss, counts = ht.balance_loss_op(X, I, E, V)
    ex = ht.Executor({'train': [loss, counts]}, ctx=ht.gpu(0), mixed_precision='bf16')
    on = np.arange(T) < T - 100
    l, c = ex.run('train', feed_dict={I: iv.astype(np.float32), V: on.astype(np.float32)}, convert_to_numpy_ret_vals=True)
    np.testing.assert_array_equal(c, np.bincount(iv[on].reshape(-1), minlength=E))


def test_choices_in_types_that_skip_whole_numbers_are_refused():
    x, idx, valid, g = _case(10, 8, 2, torch.float32, 'most', 4, 'cpu')
    for dt in (torch.bfloat16, torch.float16):
        with pytest.raises(ValueError):
            K.balance_loss(x, idx.to(dt), 8)
    for dt in (torch.float32, torch.float64, torch.int32):
        assert torch.equal(K.balance_loss(x, idx.to(dt), 8).counts, K.balance_loss(x, idx, 8).counts)
    I, V = ht.Variable(name='i', trainable=False), ht.Variable(name='v', trainable=False)
    ht.balance_loss_op(ht.Variable(name='x'), I, 8, V)
    assert I.keep_fp32                                # (what a feed under mixed precision goes by)


def test_forward_results_that_are_not_whole_are_refused():
    x, idx, valid, g = _case(10, 9, 2, torch.float32, 'most', 4, 'cpu')
    r = K.balance_loss(x, idx, 9)
    K.balance_loss_backward(x, K.BalanceLoss(r.buffer, 9), g)
    n = r.buffer.numel()
    for buffer in (r.buffer.to('meta'), r.buffer[:9], r.buffer.int(), torch.zeros(2 * n, dtype=torch.int64)[::2]):
        with pytest.raises(ValueError):
            K.balance_loss_backward(x, K.BalanceLoss(buffer, 9), g)


@pytest.mark.gpu
@pytest.mark.parametrize('T,E,k,dt,off', [
    (30001, 8, 2, torch.float32, 0), (200003, 24, 2, torch.bfloat16, 0), (100003, 60, 4, torch.bfloat16, 0),
    (100003, 60, 4, torch.float32, 1), (40001, 120, 3, torch.bfloat16, 0), (20001, 161, 6, torch.float32, 0),
    (9001, 161, 6, torch.bfloat16, 3), (70001, 256, 8, torch.bfloat16, 0), (20001, 256, 8, torch.float32, 2),
    (10001, 512, 8, torch.bfloat16, 0), (9001, 1000, 4, torch.float32, 0),
    # gradients and logits larger together than the last-level cache
    (262500, 256, 8, torch.bfloat16, 0), (140001, 240, 2, torch.float32, 0)])
def test_many_blocks_of_tokens(T, E, k, dt, off):
    """the partial sums of up to 512 blocks and every number of lanes a row, masked: values, not only that two
    calls agree"""
    wide, idx, valid, g = _case(T, E + (off and 5), k, dt, 'most', T + E, 'cuda')
    x, idx = wide[:, off:off + E], idx.clamp_max(E - 1)
    r = K.balance_loss(x, idx, E, valid)
    _check(x, idx, valid, g, r, K.balance_loss_backward(x, r, g, valid))
