"""Log probabilities of given tokens, entropy and alternatives: values and gradients against the
definition in 64 bits, on the CPU form and the HIP kernels."""
import math

import numpy as np
import pytest
import torch

import hetu_61a7_amd as ht
from hetu_61a7_amd.kernels import logprob as K

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]
U = 2.0 ** -24
INF = math.inf


def _definition(x, ids, top, grad=None, ignored=-1):
    """logp, entropy, top logp, top ids (and d logits) of fp64 rows"""
    R, V = x.shape
    x = x.double()
    valid = (ids >= 0) & (ids < V) & (ids != ignored)
    m = x.amax(1, keepdim=True)
    empty = torch.isneginf(m[:, 0])
    z = x - torch.where(torch.isneginf(m), torch.zeros_like(m), m)
    lq = z - torch.log(torch.exp(z).sum(1, keepdim=True))
    lq[empty] = -INF
    q = torch.exp(lq)
    plogp = torch.where(q > 0, q * lq, torch.zeros_like(q))
    h = -plogp.sum(1)
    logp = lq.gather(1, torch.where(valid, ids, torch.zeros_like(ids))[:, None])[:, 0]
    idx = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :top]
    tl = lq.gather(1, idx)
    z0 = torch.zeros_like(logp)
    r = [torch.where(valid, logp, z0), torch.where(valid, h, z0), torch.where(valid[:, None], tl, torch.zeros_like(tl)),
         torch.where(valid[:, None], idx, torch.full_like(idx, -1))]
    if grad is not None:
        g = grad.double()
        d = -q * (g[:, :1] + g[:, 2:].sum(1, keepdim=True)) - g[:, 1:2] * (plogp + q * h[:, None])
        for i in range(R):
            if valid[i]:
                d[i, ids[i]] += g[i, 0]
                for j in range(top):
                    d[i, idx[i, j]] += g[i, 2 + j]
        d[~valid | empty] = 0
        r += [d, torch.where(q > 0, lq, torch.zeros_like(lq)), q]
    return r


def _case(R, V, dt, mask, seed, device):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, V, generator=g) * (1 + 3 * torch.rand(R, 1, generator=g))
    ids = torch.randint(0, V, (R,), generator=g)
    low = -INF if mask == 'inf' else torch.finfo(dt).min
    if mask != 'none':
        x.masked_fill_(torch.rand(R, V, generator=g) < 0.4, low)
        x[::5] = low                                  # rows that the mask leaves empty
    if R > 2:
        ids[2::4] = -1
    return x.to(dt).to(device), ids.to(device), g


def _check(x, ids, top, dt, r, dx=None, grad=None, ignored=-1):
    """Roundings, in units U of the fp32 sums: S = sum e^d adds at most V / 256 + 64 terms one
    after another (each thread's share, then the joins), each off by |d| log2(e) + 2 roundings of
    its exponent; weighted by e^d the |d| average to at most ln V + entropy.  log S is off by that
    relative error, and the differences by a rounding of themselves."""
    V = x.shape[-1]
    x2, i2 = x.reshape(-1, V), ids.reshape(-1)
    ref = _definition(x2, i2, top, grad, ignored)
    base = U * (V / 256 + 64 + 8 * math.log(V + 1))

    def near(got, want, tol):
        want, got = want.reshape(got.shape), got.double()
        fine = torch.isfinite(want)
        assert torch.equal(torch.isfinite(got), fine) and torch.equal(got[~fine], want[~fine])
        assert bool(((got - want).abs() <= torch.as_tensor(tol, device=want.device).expand_as(want).reshape(got.shape))[fine].all())

    near(r.logp, ref[0], base + 4 * U * ref[0].abs().nan_to_num(0, 0, 0).reshape(r.logp.shape))
    near(r.entropy, ref[1], base * (2 + 2 * math.log(V + 1)))
    near(r.top_logp, ref[2], base + 4 * U * ref[2].abs().nan_to_num(0, 0, 0).reshape(r.top_logp.shape))
    assert torch.equal(r.top_ids.reshape(ref[3].shape), ref[3])
    if dx is None:
        return
    assert dx.dtype == dt and dx.shape == x.shape and dx.is_contiguous()
    d, lq, q = ref[4:]
    g = grad.double().abs()
    # p is off by (its exponent's roundings, |log p| + 4, and log S's error) of itself; it multiplies the
    # gradients, the entropy's with log p + H, whose own error is H's
    span = g[:, :1] + g[:, 2:].sum(1, keepdim=True) + g[:, 1:2] * (lq.abs() + ref[1][:, None] + 1)
    tol = q * span * (base * (3 + 2 * math.log(V + 1)) + U * (8 + 2 * top + 4 * lq.abs()))
    tol = tol + (8 + 2 * top) * U * d.abs() + 2.0 ** -126 * (1 + g.sum(1, keepdim=True))     # flushed at the least
    tol = tol + U * (4 + top) * torch.where(d.abs() > 0, (g.sum(1, keepdim=True)), torch.zeros_like(d)) * (q + (d.abs() > q * span * 1.01))
    if dt == torch.bfloat16:
        tol = tol * 1.01 + 2.0 ** -8 * d.abs()
    assert bool(((dx.reshape(d.shape).double() - d).abs() <= tol).all())


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dt', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('mask', ['none', 'inf', 'lowest'])
@pytest.mark.parametrize('R,V,top', [(1, 1, 1), (1, 2, 0), (5, 3, 3), (7, 64, 64), (9, 65, 1), (4, 257, 20), (6, 1000, 5),
                                     (3, 2049, 64), (17, 4100, 3), (2, 30522, 20), (11, 50021, 0)])
def test_values_and_gradient(R, V, top, mask, dt, device):
    x, ids, g = _case(R, V, dt, mask, 1000 * R + V, device)
    grad = torch.randn(R, 2 + top, generator=g).to(device)
    r = K.token_logprob(x, ids, top)
    dx = K.token_logprob_backward(x, ids, r, grad)
    _check(x, ids, top, dt, r, dx, grad)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dt', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('mask', ['none', 'inf', 'lowest'])
@pytest.mark.parametrize('R,V,top', [(1, 70001, 64), (6, 131072, 20), (3, 200003, 0), (128, 66000, 5), (2, 530000, 64)])
def test_few_long_rows(R, V, top, mask, dt, device):
    """at every alignment, and with fewer elements above -inf than threads"""
    if device == 'cpu' and R * V > 500000:
        pytest.skip('the CPU form has one way for every size')
    x, ids, g = _case(R, V, dt, mask, R + V, device)
    grad = torch.randn(R, 2 + top, generator=g).to(device)
    r = K.token_logprob(x, ids, top)
    _check(x, ids, top, dt, r, K.token_logprob_backward(x, ids, r, grad), grad)
    near = x.masked_fill(torch.arange(V, device=device) >= 40, -INF)
    ids = torch.where(ids >= 0, ids % 40, ids)
    _check(near, ids, min(top, 40), dt, K.token_logprob(near, ids, min(top, 40)))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dt', [torch.float32, torch.bfloat16])
def test_strided_rows_and_leading_dimensions(dt, device):
    """rows of a padded buffer at every alignment; [batch, position, V]; a transposed batch"""
    for off, V, pitch in ((0, 100, 104), (1, 999, 1003), (3, 30, 37), (5, 777, 778)):
        wide, ids, g = _case(6, pitch + off, dt, 'none', V + off, device)
        x = wide[:, off:off + V]
        ids = ids.clamp_max(V - 1)
        grad = torch.randn(6, 5, generator=g).to(device)
        r = K.token_logprob(x, ids, 3)
        _check(x, ids, 3, dt, r, K.token_logprob_backward(x, ids, r, grad), grad)
    x, ids, g = _case(6, 120, dt, 'none', 5, device)
    for x3, i3 in ((x.reshape(2, 3, 120), ids.reshape(2, 3)), (x.reshape(2, 3, 120).transpose(0, 1), ids.reshape(2, 3).t())):
        r = K.token_logprob(x3, i3, 2)
        assert r.logp.shape == i3.shape and r.top_ids.shape == i3.shape + (2,)
        grad = torch.randn(6, 4, generator=g).to(device)
        d = K.token_logprob_backward(x3, i3, r, grad.reshape(r.out.shape))
        _check(x3.reshape(-1, 120), i3.reshape(-1), 2, dt, r, d.reshape(-1, 120), grad)
    col = x.t()                                       # the vocabulary is the strided dimension
    i = torch.arange(120, device=device) % 6
    _check(col, i, 2, dt, K.token_logprob(col, i, 2))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('kind', ['equal', 'two', 'rising', 'falling', 'one thread', 'signed zero'])
def test_ties_and_adversarial_orders(kind, device):
    """equal values go to the lowest token; values that meet one thread's share alone are all found"""
    V = 70001
    x = torch.zeros(2, V)
    if kind == 'two':
        x[:, ::3] = 1.0
    elif kind == 'rising':
        x = (torch.arange(V).float() * 1e-4).repeat(2, 1)
    elif kind == 'falling':
        x = -(torch.arange(V).float() * 1e-4).repeat(2, 1)
    elif kind == 'one thread':          # 16 or 8 columns of every 2048 or 4096: many above the bound
        x = torch.randn(2, V, generator=torch.Generator().manual_seed(1)) * 0.01
        for step in (1024, 2048, 4096):
            for k in range(8):
                x[:, k::step] += 5.0
    elif kind == 'signed zero':
        x[:, 1::2] = -0.0
    for dt in (torch.float32, torch.bfloat16):
        for top in (1, 64):
            y, ids = x.to(dt).to(device), torch.tensor([0, V - 1], device=device)
            _check(y, ids, top, dt, K.token_logprob(y, ids, top))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dt', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('V', [4089, 4093, 4095, 4097, 8177, 8185, 8189, 8191, 8193, 16377])
def test_tokens_at_the_ends_of_a_row(V, dt, device):
    """the first and last tokens, given and among the alternatives, where a row ends near a block's share
    of it, at every alignment: each gets its own terms once"""
    wide, _, g = _case(33, V + 9, dt, 'none', V, device)
    wide[:, :] = wide * 0.1
    for off in range(9):
        x = wide[:, off:off + V]
        for i in (0, V - 2, V - 1):
            x[:, i] = 9.0
        ids = torch.tensor([0, V - 1, V // 2] * 11, device=device)
        grad = 1000.0 * torch.randn(33, 5, generator=g).to(device)
        r = K.token_logprob(x, ids, 3)
        _check(x, ids, 3, dt, r, K.token_logprob_backward(x, ids, r, grad), grad)


@pytest.mark.parametrize('device', DEVICES)
def test_rows_that_are_not_read(device):
    """ignored and out-of-range tokens: NaN and infinities in their rows reach nothing"""
    V = 500
    x, ids, g = _case(8, V, torch.float32, 'none', 3, device)
    ids = torch.tensor([3, -1, V, 7, -100, 9, 2 ** 40, 7], device=device)
    x[[1, 2, 4, 6]] = float('nan')
    grad = torch.randn(8, 4, generator=g).to(device)
    r = K.token_logprob(x, ids, 2, ignored_index=9)
    d = K.token_logprob_backward(x, ids, r, grad, ignored_index=9)
    _check(x.nan_to_num(0), ids, 2, torch.float32, r, d, grad, ignored=9)
    for i in (1, 2, 4, 5, 6):
        assert not r.out[i].any() and bool((r.top_ids[i] == -1).all()) and not d[i].any()


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('what', [float('nan'), INF])
def test_nan_and_inf_make_their_row_nan(what, device):
    x, ids, g = _case(3, 3000, torch.float32, 'none', 4, device)
    ids[:] = 5
    clean = x.clone()
    x[1, 2222] = what
    grad = torch.randn(3, 4, generator=g).to(device)
    r = K.token_logprob(x, ids, 2)
    d = K.token_logprob_backward(x, ids, r, grad)
    assert bool(r.logp[1].isnan()) and bool(r.entropy[1].isnan()) and bool(d[1].isnan().all())
    assert bool(((r.top_ids[1] >= 0) & (r.top_ids[1] < 3000)).all())
    keep = torch.tensor([0, 2], device=device)
    c = K.token_logprob(clean, ids, 2)
    assert torch.equal(r.out[keep], c.out[keep])
    assert torch.equal(d[keep], K.token_logprob_backward(clean, ids, c, grad)[keep])


@pytest.mark.parametrize('device', DEVICES)
def test_gradient_against_differences(device):
    """d (sum of g * out) by central differences of the values in 64 bits"""
    x, ids, g = _case(2, 40, torch.float32, 'none', 7, device)
    ids[:] = torch.tensor([4, 39])
    grad = torch.randn(2, 5, generator=g).to(device)
    r = K.token_logprob(x, ids, 3)
    d = K.token_logprob_backward(x, ids, r, grad).double()
    h = 1e-5

    def value(y):
        a = _definition(y, ids, 3)
        return float((torch.cat([a[0][:, None], a[1][:, None], a[2]], 1) * grad.double()).sum())
    for i in range(2):
        for j in range(0, 40, 3):
            a, b = x.double().clone(), x.double().clone()
            a[i, j] += h
            b[i, j] -= h
            assert abs((value(a) - value(b)) / (2 * h) - float(d[i, j])) < 1e-6   # h^2 and 1e-16 / h, fp32's U


@pytest.mark.parametrize('device', DEVICES)
def test_integer_types_and_no_rows(device):
    x, ids, _ = _case(4, 50, torch.float32, 'none', 8, device)
    want = K.token_logprob(x, ids, 1)
    for t in (ids.int(), ids.float()):
        assert torch.equal(K.token_logprob(x, t, 1).out, want.out)
    r = K.token_logprob(x[:0], ids[:0], 1)
    assert r.out.shape == (0, 3) and r.top_ids.shape == (0, 1)
    assert K.token_logprob_backward(x[:0], ids[:0], r, r.out).shape == (0, 50)
    one = K.token_logprob(x[0], ids[0], 1)            # a single row without a leading dimension
    assert one.logp.shape == () and torch.equal(one.out, want.out[0])


def test_refusals():
    x, ids, _ = _case(4, 50, torch.float32, 'none', 9, 'cpu')
    for a in ((x.double(), ids, 0), (x.half(), ids, 0), (x, ids[:3], 0), (x, ids, -1), (x, ids, 51), (x, ids, 65),
              (x[:, :0], ids, 0), (x, ids.to(torch.bfloat16), 0)):
        with pytest.raises(ValueError):
            K.token_logprob(*a)
    big = torch.zeros(1, 100)
    with pytest.raises(ValueError):
        K.token_logprob(big, torch.zeros(1, dtype=torch.int64), 65)
    r = K.token_logprob(x, ids, 2)
    for a in ((x, ids, r, torch.zeros(4, 3)), (x[:2], ids[:2], r, torch.zeros(2, 4)), (x[:, :1], ids, r, torch.zeros(4, 4))):
        with pytest.raises(ValueError):
            K.token_logprob_backward(*a)
    with pytest.raises(ValueError):
        ht.token_logprob_op(ht.Variable(name='x'), ht.Variable(name='i'), top=65)


@pytest.mark.gpu
def test_same_call_gives_the_same_bits_and_another_stream():
    from hetu_61a7_amd import runtime as RT
    x, ids, g = _case(64, 30522, torch.bfloat16, 'none', 10, 'cuda')
    grad = torch.randn(64, 22, generator=g).to('cuda')
    r = K.token_logprob(x, ids, 20)
    d = K.token_logprob_backward(x, ids, r, grad)
    s = RT.DeviceStream()
    s.wait_stream(None)
    with RT.use_stream(s):
        r2 = K.token_logprob(x, ids, 20)
        d2 = K.token_logprob_backward(x, ids, r2, grad)
    torch.cuda.synchronize()
    assert torch.equal(r.out, r2.out) and torch.equal(r.top_ids, r2.top_ids) and torch.equal(d, d2)


@pytest.mark.gpu
def test_more_rows_than_one_dimension_of_a_launch_holds():
    """2^24 + 5 rows of 3 logits: 2^32 threads in the backward pass"""
    R = (1 << 24) + 5
    x = torch.randn(R, 3, device='cuda').to(torch.bfloat16)
    ids = torch.arange(R, device='cuda') % 3
    grad = torch.ones(R, 2, device='cuda')
    grad[:, 1] = 0
    r = K.token_logprob(x, ids)
    d = K.token_logprob_backward(x, ids, r, grad)
    for a, b in ((0, 1000), ((1 << 20) - 500, (1 << 20) + 500), ((1 << 24) - 500, R)):
        s = slice(a, b)
        part = K.TokenLogProb(r.buffer[s], None)
        _check(x[s], ids[s], 0, torch.bfloat16, part, d[s], grad[s])


# ---- as graph operators ------------------------------------------------------------------------
@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('graph', [False, True])
def test_op_values_and_gradients(device, graph):
    """every column's gradient reaches the logits in one pass; the step is replayed when captured"""
    if graph and device == 'cpu':
        pytest.skip('no captured steps on the CPU')
    R, V, top = 12, 301, 3
    x, ids, g = _case(R, V, torch.float32, 'none', 11, 'cpu')
    w = torch.randn(R, 2 + top, generator=g)
    X = ht.Variable(name='x', value=x.numpy())
    I = ht.Variable(name='ids', trainable=False)
    c = [ht.Variable(name='c%d' % i, trainable=False) for i in range(3)]
    logp, ent, tl, ti = ht.token_logprob_op(X, I, top=top)
    loss = ht.reduce_sum_op(logp * c[0], [0]) + ht.reduce_sum_op(ent * c[1], [0]) + \
        ht.reduce_sum_op(ht.reduce_sum_op(tl * c[2], [1]), [0])
    (gx,) = ht.gradients(loss, [X])
    ex = ht.Executor({'train': [logp, ent, tl, ti, gx]}, ctx=ht.cpu(0) if device == 'cpu' else ht.gpu(0), use_hipgraph=graph)
    feed = {I: ids.numpy().astype(np.float32), c[0]: w[:, 0].numpy(), c[1]: w[:, 1].numpy(), c[2]: w[:, 2:].numpy()}
    for _ in range(6 if graph else 1):
        out = ex.run('train', feed_dict=feed, convert_to_numpy_ret_vals=True)
        lp, e, t, i, d = [torch.from_numpy(np.asarray(o)) for o in out]
        r = K.TokenLogProb(torch.cat([lp[:, None], e[:, None], t, t[:, :2]], 1), i)
        _check(x, ids, top, torch.float32, r, d, w)


@pytest.mark.parametrize('device', DEVICES)
def test_op_without_alternatives(device):
    x, ids, _ = _case(6, 90, torch.float32, 'none', 12, 'cpu')
    X, I = ht.Variable(name='x', value=x.numpy()), ht.Variable(name='ids', trainable=False)
    logp, ent = ht.token_logprob_op(X, I)
    loss = ht.reduce_mean_op(logp, [0])
    (gx,) = ht.gradients(loss, [X])
    ex = ht.Executor({'train': [logp, gx]}, ctx=ht.cpu(0) if device == 'cpu' else ht.gpu(0))
    lp, d = ex.run('train', feed_dict={I: ids.numpy()}, convert_to_numpy_ret_vals=True)
    grad = torch.zeros(6, 2)
    grad[:, 0] = 1.0 / 6
    r = K.token_logprob(x, ids)
    _check(x, ids, 0, torch.float32, r, torch.from_numpy(d), grad)
    np.testing.assert_allclose(lp, r.logp.numpy(), rtol=1e-6, atol=1e-6)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dt,V', [(torch.float32, 4097), (torch.float32, 9001), (torch.bfloat16, 9001), (torch.bfloat16, 20011)])
def test_ties_with_the_first_elements_of_an_unaligned_row(dt, V, device):
    """a row's first elements, up to its first 16-byte border, are taken apart from the rest: where they tie with
    later ones, the lowest token still wins, at every alignment and for both sizes of a block"""
    n = 16 // torch.empty((), dtype=dt).element_size()
    threads = 1024 if V * (16 // n) >= 32768 else 256
    g = torch.Generator().manual_seed(V)
    for off in range(1, n):
        wide = torch.full((4, -(-(V + off) // n) * n), -3.0)
        for row, head in enumerate((0, n - off - 1, 0, 0)):
            # the first elements, a thread far behind, and the first threads' second share alone
            ties = [off + head, n * 101 + 3, n * (1 + threads), n * (2 + threads), n * (3 + threads), n * (4 + threads)]
            wide[row, ties[:3] if row < 2 else ties] = 2.0
            if row == 3:
                wide[row, 5 * n::7] = 2.0
        x = wide.to(dt).to(device)[:, off:off + V]
        ids = torch.zeros(4, dtype=torch.int64, device=device)
        for top in (1, 2, 3, 20, 40):
            _check(x, ids, top, dt, K.token_logprob(x, ids, top))
        whole = torch.randint(0, 7, (40, wide.shape[1]), generator=g).float().to(dt).to(device)[:, off:off + V]
        whole[:, 0] = torch.where(torch.arange(40, device=device) % 2 == 0, 6.0, 0.0).to(dt)
        whole[::2, 5:whole.shape[1] // 2] = 1.0
        ids = torch.zeros(40, dtype=torch.int64, device=device)
        for top in (1, 20, 64):
            _check(whole, ids, top, dt, K.token_logprob(whole, ids, top))


@pytest.mark.gpu
def test_gradient_of_the_longest_row_at_another_alignment():
    """2^31 - 65 logits of a row that starts one element off the gradient's alignment: the last elements'
    numbers plus a block's threads pass 31 bits"""
    V = 2 ** 31 - 65
    x = torch.zeros(V + 1, dtype=torch.bfloat16, device='cuda')[1:]
    x[V - 3] = 20.0
    ids = torch.tensor([V - 1], device='cuda')
    r = K.token_logprob(x[None], ids)
    # S = (V - 1) e^-20 + 1: a thread adds 2^21 terms one after another, of which each sum of 32 is one
    lse = 20.0 + math.log1p((V - 1) * math.exp(-20.0))
    slack = U * (2 ** 21 / 32 + 200)
    assert abs(float(r.logp[0]) + lse) <= slack + 4 * U * lse
    d = K.token_logprob_backward(x[None], ids, r, torch.tensor([[1.0, 0.0]], device='cuda'))[0]
    p = math.exp(-lse)
    step = 2.0 ** -8 + 2 * slack + 40 * U
    for a, b in ((0, 3000), (V // 2, V // 2 + 3000), (V - 3000, V - 3)):
        assert bool(((d[a:b].double() + p).abs() <= step * p).all())
    assert bool(((d[3000:V - 3000:4099].double() + p).abs() <= step * p).all())
    want = torch.tensor([-math.exp(20.0) * p, -p, 1.0 - p], dtype=torch.float64, device='cuda')
    assert bool(((d[V - 3:].double() - want).abs() <= step * want.abs()).all())


def test_forward_results_that_are_not_whole_are_refused():
    """of another device, strided, or without their ids: the backward pass would read where nothing is"""
    x, ids, _ = _case(4, 50, torch.float32, 'none', 9, 'cpu')
    grad, r = torch.zeros(4, 4), K.token_logprob(x, ids, 2)
    K.token_logprob_backward(x, ids, K.TokenLogProb(r.buffer, r.ids), grad)
    wide = torch.zeros(4, 12)
    for buffer, tokens in ((r.buffer.to('meta'), r.ids), (r.buffer, r.ids.to('meta')), (r.buffer, None), (wide[:, ::2], r.ids),
                           (r.buffer, torch.zeros(4, 4, dtype=torch.int64)[:, ::2]), (r.buffer, r.ids[:2]),
                           (r.buffer, r.ids.int()), (r.buffer.double(), r.ids)):
        with pytest.raises(ValueError):
            K.token_logprob_backward(x, ids, K.TokenLogProb(buffer, tokens), grad)


@pytest.mark.gpu
@pytest.mark.parametrize('R,V,pitch,top,dt', [
    # gradients beyond half the last-level cache, then logits beyond three times it
    (1101, 61003, 61003, 0, torch.bfloat16), (1101, 61003, 61004, 3, torch.bfloat16), (600, 60001, 60001, 3, torch.float32),
    (600, 60001, 60003, 0, torch.float32), (6700, 60103, 60103, 2, torch.bfloat16), (6700, 60103, 60112, 0, torch.bfloat16),
    (3400, 60001, 60001, 0, torch.float32), (3400, 60001, 60002, 2, torch.float32)])
def test_gradients_larger_than_the_cache(R, V, pitch, top, dt):
    """rows aligned like the gradient's (pitch = V) and not, of the sizes where the gradient, then the logits too,
    go past the last-level cache: rows at both ends and between against 64 bits"""
    g = torch.Generator(device='cuda').manual_seed(R + pitch)
    x = torch.empty(R, pitch, dtype=dt, device='cuda')
    for a in range(0, R, 500):
        x[a:a + 500] = (2 * torch.randn(min(500, R - a), pitch, generator=g, device='cuda')).to(dt)
    x = x[:, pitch - V:]
    ids = torch.randint(0, V, (R,), generator=g, device='cuda')
    ids[2::4] = -1
    x[5] = -INF
    grad = torch.randn(R, 2 + top, generator=g, device='cuda')
    r = K.token_logprob(x, ids, top)
    d = K.token_logprob_backward(x, ids, r, grad)
    rows = torch.unique(torch.cat([torch.arange(8), torch.arange(R - 8, R), torch.linspace(8, R - 9, 16).long()])).cuda()
    part = K.TokenLogProb(r.buffer[rows], r.ids[rows] if top else None)
    _check(x[rows], ids[rows], top, dt, part, d[rows], grad[rows])
    # every row: its gradient's sum is 0 but for the roundings of its elements, each at most half a step of
    # bf16 of itself, and zero for tokens that are not there
    eps = 2.0 ** -8 if dt == torch.bfloat16 else 2.0 ** -20
    for a in range(0, R, 500):
        part = d[a:a + 500].double()
        assert bool((part.sum(1).abs() <= eps * part.abs().sum(1) + 1e-5 * grad[a:a + 500].double().abs().sum(1)).all())
        assert not part[ids[a:a + 500] < 0].any()
