"""Soft correspondence (soft_match, its gradients, TemplateStore) against a plain implementation in 64 bits.

Tolerances count roundings, relative to the root mean square (or, where larger, the value):
  float32   dot products of C terms and sums of n weights accumulate about sqrt(C + n) / 2 half steps of 2^-24 of their
            terms, the exponent |z| <= 60 adds |z| 2^-24 to a weight: 2^-24 (60 + 60) = 7e-6, taken as 2e-5.
  bfloat16  inputs are taken as they are; one rounding of a weight (2^-9 on average, 2^-8 at most) and one of the result
            (2^-8 at most): 2^-7 of the value where the weights' roundings do not cancel, taken per element against
            2^-7 (|out| + sum_j P |v|); a gradient passes one more rounded product: 3 x 2^-8 of the sum of magnitudes.
"""
import math

import numpy as np
import pytest
import torch

gpu = pytest.mark.gpu
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def sc():
    from pose_estimation_amd import soft_correspondence
    return soft_correspondence


# ------------------------------------------------------------------------------------------------ the oracle
def oracle(q, r, v, heads, scale, cap=0.0, falloff=None, xy=None, width=None, mask=None, count=None, d_out=None, d_lse=None):
    """numpy float64; q (b,C,n), r (b,C,m), v (b,Cv,m).  Returns out, lse, the magnitude sum_j P |v| and, with d_out, the
    gradients with the sums of magnitudes that their roundings go by."""
    q, r, v = (np.asarray(x, np.float64) for x in (q, r, v))
    b, c, n = q.shape
    m, cv = r.shape[2], v.shape[1]
    d, e = c // heads, cv // heads
    out, lse, mag = np.zeros((b, cv, n)), np.full((b, heads, n), -np.inf), np.zeros((b, cv, n))
    dq, dr, dv = np.zeros_like(q), np.zeros_like(r), np.zeros_like(v)
    mq, mr, mv = np.zeros_like(q), np.zeros_like(r), np.zeros_like(v)
    for i in range(b):
        live = n if count is None else int(min(max(count[i], 0), n))
        js = np.arange(m) if mask is None else np.flatnonzero(np.asarray(mask[i]).reshape(-1))
        if live == 0 or js.size == 0:
            continue
        for h in range(heads):
            a, w = slice(h * d, h * d + d), slice(h * e, h * e + e)
            qq, rr, vv = q[i, a, :live], r[i, a][:, js], v[i, w][:, js]
            x = scale * qq.T @ rr
            t = np.tanh(x / cap) if cap else None
            z = cap * t if cap else x
            if falloff is not None:
                place = xy[i, :live] if xy is not None else np.stack([np.arange(live) % width, np.arange(live) // width], 1)
                cell = np.stack([js % width, js // width], 1)
                z = z - falloff[h] * ((place[:, None] - cell[None]) ** 2).sum(2)
            top = z.max(1, keepdims=True)
            p = np.exp(z - top)
            lse[i, h, :live] = np.log(p.sum(1)) + top[:, 0]
            p /= p.sum(1, keepdims=True)
            out[i, w, :live] = vv @ p.T
            mag[i, w, :live] = np.abs(vv) @ p.T
            if d_out is None:
                continue
            do = np.asarray(d_out, np.float64)[i, w, :live]
            dp = do.T @ vv
            delta = (p * dp).sum(1, keepdims=True)
            g = p * (dp - delta + (0 if d_lse is None else np.asarray(d_lse, np.float64)[i, h, :live, None]))
            # a rounded product dp (float32) and delta: their errors go by magnitudes
            size = p * (np.abs(dp) + (p * np.abs(dp)).sum(1, keepdims=True) + (0 if d_lse is None else np.abs(np.asarray(d_lse, np.float64)[i, h, :live, None])))
            slope = scale * (1 - t * t) if cap else scale
            g, size = g * slope, size * np.abs(slope)
            dq[i, a, :live] = rr @ g.T
            mq[i, a, :live] = np.abs(rr) @ size.T
            dr[i, a][:, js] += qq @ g
            mr[i, a][:, js] += np.abs(qq) @ size
            dv[i, w][:, js] += do @ p
            mv[i, w][:, js] += np.abs(do) @ p
    return out, lse, mag, (dq, dr, dv), (mq, mr, mv)


def rand(seed, shape, dtype, unit=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g)
    if unit:
        x = x / x.square().sum(1, keepdim=True).sqrt()
    return x.to(dtype)


def host(x):
    return x.detach().double().cpu().numpy()


def flat(x):
    return host(x).reshape(tuple(x.shape[:2]) + (-1,))


def near(got, want, mag, dtype, roundings):
    """|got - want| within `roundings` bfloat16 half steps of the sum of magnitudes, or 2e-5 of it in float32, plus the
    rounding of the result itself."""
    got = flat(got) if got.dim() > 2 else host(got)
    part = roundings * HALF[dtype] if dtype == BF16 else 2e-5
    assert np.isfinite(got).all()
    err = np.abs(got - want) - (part * mag + HALF[dtype] * np.abs(want) + 1e-30)
    assert err.max(initial=-1) <= 0, float(err.max())


def near_lse(got, want):
    got = host(got)
    assert np.array_equal(np.isneginf(got), np.isneginf(want))
    ok = np.isfinite(want)
    # the log of a float32 sum: 2^-24 sqrt(n) of the sum, and |z| 2^-24 of the score
    assert np.abs(got[ok] - want[ok]).max(initial=0) <= 2e-5 * max(1.0, np.abs(want[ok]).max(initial=0))


def inputs(dtype, b, c, grid, n=0, cv=0, seed=0):
    h, w = grid
    q = rand(seed + 1, (b, c, n) if n else (b, c, h, w), dtype)
    r = rand(seed + 2, (b, c, h, w), dtype)
    v = rand(seed + 3, (b, cv, h, w), dtype, unit=False) if cv else None
    return q, r, v


def silhouette(seed, b, h, w, share=0.6):
    g = torch.Generator().manual_seed(seed)
    return torch.rand((b, h, w), generator=g) < share


def cuda(*xs):
    return [x.cuda() if x is not None else None for x in xs]


SHAPES = [  # batch, channels, heads, value channels, grid, queries (0: the grid)
    (1, 128, 1, 0, (28, 28), 10),
    (2, 64, 2, 0, (1, 1), 1),
    (1, 32, 1, 2, (7, 9), 0),
    (2, 100, 2, 36, (13, 11), 33),
    (1, 3, 1, 1, (5, 64), 129),
    (1, 256, 1, 0, (8, 9), 65),
    (1, 40, 1, 200, (16, 16), 31),
    (2, 128, 1, 128, (32, 33), 0),
    (1, 130, 1, 0, (12, 12), 0),
    (1, 64, 1, 0, (3, 21), 64),
]


# ------------------------------------------------------------------------------------------------ forward
@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_shapes(sc, dtype, shape):
    b, c, heads, cv, grid, n = shape
    q, r, v = inputs(dtype, b, c, grid, n, cv)
    out, lse = sc.soft_match(*cuda(q, r, v), heads=heads, scale=12.0, return_lse=True)
    assert out.dtype == dtype and out.shape == (b, cv or c) + tuple(q.shape[2:]) and lse.shape == (b, heads, flat(q).shape[2])
    want = oracle(flat(q), flat(r), flat(r if v is None else v), heads, 12.0)
    near(out, want[0], want[2], dtype, 1)
    near_lse(lse, want[1])


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [0, 5, 77])
@pytest.mark.parametrize("cap, falloff, masked", [(0.0, None, True), (8.0, None, False), (0.0, 0.03, False), (5.0, 0.1, True)])
def test_forward_scores(sc, dtype, n, cap, falloff, masked):
    b, c, heads, grid = 3, 48, 2, (15, 17)
    q, r, v = inputs(dtype, b, c, grid, n, 64, seed=5)
    mask = silhouette(1, b, *grid) if masked else None
    if masked:
        mask[1] = False                                  # an item without a cell
    fall = torch.tensor([falloff, 2 * falloff]) if falloff else None
    xy = torch.rand((b, n, 2), generator=torch.Generator().manual_seed(2)) * 14 if n else None
    count = torch.tensor([q.shape[2] if n else 255, 3, 0], dtype=torch.int32)
    out, lse = sc.soft_match(*cuda(q, r, v), heads=heads, scale=30.0, cap=cap, falloff=fall, query_xy=xy if falloff else None,
                             mask=mask.cuda() if masked else None, num_query=count.cuda(), return_lse=True)
    want = oracle(flat(q), flat(r), flat(v), heads, 30.0, cap, None if fall is None else fall.double().numpy(),
                  None if xy is None else xy.double().numpy(), grid[1], None if mask is None else mask.numpy(), count.numpy())
    near(out, want[0], want[2], dtype, 1)
    near_lse(lse, want[1])
    assert (flat(out)[2] == 0).all() and np.isneginf(host(lse)[2]).all()


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
def test_masked_cells_may_hold_anything(sc, dtype, bad):
    grid = (9, 15)
    q, r, v = inputs(dtype, 1, 32, grid, 0, 32, seed=9)
    mask = silhouette(3, 1, *grid, share=0.5)
    opts = dict(scale=9.0, cap=4.0, mask=mask.cuda())
    want = sc.soft_match(*cuda(q, r, v), **opts)
    r2, v2 = (torch.where(mask[:, None], x, torch.full_like(x, bad)) for x in (r, v))
    leaves = [x.requires_grad_() for x in cuda(q, r2, v2)]
    got = sc.soft_match(*leaves, **opts)
    assert torch.equal(got, want)
    grads = torch.autograd.grad(got, leaves, torch.ones_like(got))
    clean = [x.requires_grad_() for x in cuda(q, r, v)]
    for g, w in zip(grads, torch.autograd.grad(sc.soft_match(*clean, **opts), clean, torch.ones_like(got))):
        assert torch.equal(g, w)


@gpu
def test_strides_orders_and_arrays(sc):
    q, r, v = inputs(F32, 2, 24, (10, 6), 0, 16, seed=3)
    want = sc.soft_match(*cuda(q, r, v), scale=5.0)
    last = [x.cuda().to(memory_format=torch.channels_last) for x in (q, r, v)]
    assert torch.equal(sc.soft_match(*last, scale=5.0), want)
    assert torch.equal(sc.soft_match(q.cuda()[:, :, :, ::2], *cuda(r, v), scale=5.0), want[:, :, :, ::2])
    # a batch-shared template
    shared = sc.soft_match(q.cuda(), r.cuda()[:1].expand(2, -1, -1, -1), v.cuda()[:1].expand(2, -1, -1, -1), scale=5.0)
    assert torch.equal(shared[0], want[0])
    # a view that starts off the 16-byte grid
    odd = torch.empty(r.numel() + 1, device="cuda")[1:].view(r.shape).copy_(r)
    assert torch.equal(sc.soft_match(q.cuda(), odd, v.cuda(), scale=5.0), want)
    arr = sc.soft_match(q.numpy(), r.numpy(), v.numpy(), scale=5.0)
    assert isinstance(arr, np.ndarray) and np.array_equal(arr, want.cpu().numpy())
    empty = sc.soft_match(torch.empty((2, 24, 0), device="cuda"), *cuda(r, v), scale=5.0, return_lse=True)
    assert empty[0].shape == (2, 16, 0) and empty[1].shape == (2, 1, 0)


@gpu
def test_bfloat16_view_at_an_odd_address(sc):
    q, r, _ = inputs(BF16, 1, 64, (9, 13), 40, seed=4)
    want = sc.soft_match(*cuda(q, r), scale=9.0)
    odd = torch.empty(r.numel() + 1, dtype=BF16, device="cuda")[1:].view(r.shape).copy_(r)
    assert torch.equal(sc.soft_match(q.cuda(), odd, scale=9.0), want)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_peaked_match_is_the_nearest_neighbour(sc, dtype):
    """At a large scale the soft match returns the features of dense_nn's nearest cell."""
    from pose_estimation_amd import correspondence
    r = rand(1, (2, 64, 12, 12), dtype).cuda()
    at = torch.randint(144, (2, 30), generator=torch.Generator().manual_seed(0)).cuda()
    q = r.flatten(2).gather(2, at[:, None].expand(2, 64, 30))
    _, ind = correspondence.dense_nn(q, r, 1)
    out = sc.soft_match(q, r, scale=400.0)
    want = r.flatten(2).gather(2, (ind.long() - 1).expand(2, 64, 30))
    # the runner-up lies a cosine of at least 0.3 lower: its weight is below exp(-120)
    assert torch.allclose(out.float(), want.float(), rtol=2 * HALF[dtype], atol=1e-6)


@gpu
def test_large_scores_do_not_overflow(sc):
    q, r, v = inputs(F32, 1, 16, (6, 6), 0, 4, seed=8)
    for scale in (3e4, -3e4):
        out, lse = sc.soft_match(*cuda(q, r, v), scale=scale, return_lse=True)
        want = oracle(flat(q), flat(r), flat(v), 1, scale)
        # scores of 3e4 carry 3e4 2^-24 = 2e-3 of absolute error into the weights
        assert torch.isfinite(out).all() and np.abs(flat(out) - want[0]).max() <= 8e-3 * np.abs(want[2]).max()
        assert np.allclose(host(lse), want[1], rtol=1e-6)


# ------------------------------------------------------------------------------------------------ backward
def gradients(sc, q, r, v, d_out, d_lse, **opts):
    leaves = [x.detach().requires_grad_() for x in (q, r, v) if x is not None]
    out, lse = sc.soft_match(*leaves, return_lse=True, **opts)
    outs, gos = ([out, lse], [d_out, d_lse]) if d_lse is not None else ([out], [d_out])
    return out, torch.autograd.grad(outs, leaves, gos)


def check_gradients(got, want, dtype, shared):
    (dq, dr, dv), (mq, mr, mv) = want[3], want[4]
    near(got[0], dq, mq, dtype, 3)
    if shared:
        near(got[1], dr + dv, mr + mv, dtype, 3)
    else:
        near(got[1], dr, mr, dtype, 3)
        near(got[2], dv, mv, dtype, 3)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", SHAPES)
def test_backward_shapes(sc, dtype, shape):
    b, c, heads, cv, grid, n = shape
    q, r, v = inputs(dtype, b, c, grid, n, cv, seed=20)
    d_out = rand(30, (b, cv or c) + tuple(q.shape[2:]), dtype, unit=False)
    out, got = gradients(sc, *cuda(q, r, v, d_out), None, heads=heads, scale=12.0)
    want = oracle(flat(q), flat(r), flat(r if v is None else v), heads, 12.0, d_out=flat(d_out))
    check_gradients(got, want, dtype, v is None)
    near(out, want[0], want[2], dtype, 1)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [0, 40])
@pytest.mark.parametrize("cap, falloff, masked", [(0.0, None, True), (8.0, None, False), (0.0, 0.03, False), (5.0, 0.1, True)])
def test_backward_scores(sc, dtype, n, cap, falloff, masked):
    b, c, heads, grid = 3, 48, 2, (15, 17)
    q, r, v = inputs(dtype, b, c, grid, n, 64, seed=40)
    nq = n or 255
    mask = silhouette(1, b, *grid) if masked else None
    if masked:
        mask[1] = False
    fall = torch.tensor([falloff, 2 * falloff]) if falloff else None
    xy = torch.rand((b, n, 2), generator=torch.Generator().manual_seed(2)) * 14 if n else None
    count = torch.tensor([nq, 3, 20], dtype=torch.int64)
    d_out = rand(31, (b, 64) + tuple(q.shape[2:]), dtype, unit=False)
    d_lse = rand(32, (b, heads, nq), F32, unit=False)
    q[2].view(c, -1)[:, 20:] = float("nan")              # what lies behind the real queries is not read
    d_out[2].view(64, -1)[:, 20:] = float("nan")
    _, got = gradients(sc, *cuda(q, r, v, d_out, d_lse), heads=heads, scale=30.0, cap=cap, falloff=fall,
                       query_xy=xy if falloff else None, mask=mask.cuda() if masked else None, num_query=count.cuda())
    want = oracle(flat(q), flat(r), flat(v), heads, 30.0, cap, None if fall is None else fall.double().numpy(),
                  None if xy is None else xy.double().numpy(), grid[1], None if mask is None else mask.numpy(), count.numpy(),
                  flat(d_out), host(d_lse))
    check_gradients(got, want, dtype, False)
    assert (flat(got[0])[2][:, 20:] == 0).all()
    if masked:
        assert (flat(got[1])[1] == 0).all() and (flat(got[2])[~np.broadcast_to(mask.flatten(1).numpy()[:, None], (b, 64, 255))] == 0).all()


@gpu
def test_gradient_against_differences(sc):
    """Central differences of the float32 forward along random directions."""
    q, r, v = cuda(*inputs(F32, 1, 16, (5, 6), 0, 8, seed=50))
    opts = dict(scale=4.0, cap=3.0, falloff=0.05)
    d_out, d_lse = rand(51, (1, 8, 5, 6), F32, unit=False).cuda(), rand(52, (1, 1, 30), F32, unit=False).cuda()
    _, grads = gradients(sc, q, r, v, d_out, d_lse, **opts)

    def loss(*x):
        out, lse = sc.soft_match(*x, return_lse=True, **opts)
        return float((out.double() * d_out).sum() + (lse.double() * d_lse).sum())

    for i, x in enumerate((q, r, v)):
        u = rand(60 + i, tuple(x.shape), F32, unit=False).cuda()
        step = 2.0 ** -6
        args = lambda s: [y + s * u if j == i else y for j, y in enumerate((q, r, v))]
        slope = (loss(*args(step)) - loss(*args(-step))) / (2 * step)
        # third-order term: step^2 / 6 times the third derivative (scores change by up to 4 |u| step: below 2e-3 here),
        # and forward errors of 2e-5 * 30 / (2 step) = 2e-2 at the very most
        want = float((grads[i].double() * u).sum())
        assert abs(slope - want) <= 3e-2 * max(1.0, abs(want)), (i, slope, want)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_only_the_wanted_gradients(sc, dtype):
    q, r, v = cuda(*inputs(dtype, 2, 32, (6, 7), 0, 16, seed=70))
    d_out = torch.ones((2, 16, 6, 7), dtype=dtype, device="cuda")
    _, want = gradients(sc, q, r, v, d_out, None, scale=5.0)
    v1 = v.detach().requires_grad_()
    sc.soft_match(q, r, v1, scale=5.0).backward(d_out)
    assert torch.equal(v1.grad, want[2])
    # the confidence alone
    q1 = q.detach().requires_grad_()
    _, lse = sc.soft_match(q1, r, v, scale=5.0, return_lse=True)
    lse.sum().backward()
    z = np.zeros((2, 16, 42))
    ref = oracle(flat(q), flat(r), flat(v), 1, 5.0, d_out=z, d_lse=np.ones((2, 1, 42)))
    near(q1.grad, ref[3][0], ref[4][0], dtype, 3)
    # a template shared by the batch: its gradient is the sum over the items
    r1 = r[:1].detach().requires_grad_()
    sc.soft_match(q, r1.expand(2, -1, -1, -1), v, scale=5.0).backward(d_out)
    ref = oracle(flat(q), flat(r[:1].expand(2, -1, -1, -1)), flat(v), 1, 5.0, d_out=flat(d_out))
    near(r1.grad, ref[3][1].sum(0, keepdims=True), 2 * ref[4][1].sum(0, keepdims=True), dtype, 3)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("c, cv", [(32, 0), (32, 16), (128, 0), (256, 256)])
def test_gradients_without_queries(sc, dtype, c, cv):
    """An item set without a single query: its template gets zeros."""
    for grid in ((3, 5), (20, 24)):
        q, r, v = cuda(*inputs(dtype, 2, c, grid, 0, cv, seed=75))
        q = q.flatten(2)[:, :, :0]
        leaves = [x.detach().requires_grad_() for x in (q, r, v) if x is not None]
        out, lse = sc.soft_match(*leaves, scale=5.0, return_lse=True)
        got = torch.autograd.grad([out, lse], leaves, [torch.ones_like(out), torch.ones_like(lse)])
        assert out.shape == (2, cv or c, 0) and lse.shape == (2, 1, 0) and got[0].shape == q.shape
        for g, x in zip(got[1:], leaves[1:]):
            assert g.shape == x.shape and g.dtype == dtype and (g == 0).all()


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_runs_agree_bit_for_bit(sc, dtype):
    q, r, v = cuda(*inputs(dtype, 2, 128, (28, 28), 50, 0, seed=80))
    d_out = rand(81, (2, 128, 50), dtype, unit=False).cuda()
    first = gradients(sc, q, r, v, d_out, None, scale=15.0)
    for _ in range(3):
        again = gradients(sc, q, r, v, d_out, None, scale=15.0)
        assert torch.equal(first[0], again[0]) and all(torch.equal(a, b) for a, b in zip(first[1], again[1]))


@gpu
def test_changed_mask_is_noticed(sc):
    q, r, _ = cuda(*inputs(F32, 1, 8, (4, 4)))
    mask = torch.ones((1, 4, 4), dtype=torch.bool, device="cuda")
    q.requires_grad_()
    out = sc.soft_match(q, r, mask=mask)
    mask[0, 0, 0] = False
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


@gpu
def test_maps_beyond_32_bit_offsets(sc):
    """The last of 9 items lies more than 2^31 numbers into the maps.  Its queries are cells of the map, so that one weight is
    nearly 1 and its dP - Delta cancels: the errors go by the magnitudes before that, as everywhere here."""
    b, c, h, scale = 9, 256, 1024, 25.0
    g = torch.Generator(device="cuda").manual_seed(210)
    r = torch.empty((b, c, h, h), dtype=BF16, device="cuda")
    for i in range(b):
        x = torch.randn((c, h, h), generator=g, device="cuda")
        r[i] = x / x.square().sum(0).sqrt()
    at = torch.randint(h * h, (5,), generator=g, device="cuda")
    q = r.flatten(2)[:, :, at].contiguous()
    d_out = torch.randn(q.shape, generator=g, device="cuda").to(BF16)
    out, (dq, dr) = gradients(sc, q, r, None, d_out, None, scale=scale)
    out, dq, dr = (x[-1].detach().flatten(1).double() for x in (out, dq, dr))
    q, r, d = (x[-1].flatten(1).double() for x in (q, r, d_out))
    p = torch.softmax(scale * q.T @ r, 1)
    dp = d.T @ r
    dx = scale * p * (dp - (p * dp).sum(1, keepdim=True))
    size = scale * p * (dp.abs() + (p * dp.abs()).sum(1, keepdim=True))
    for got, want, mag, roundings in ((out, r @ p.T, r.abs() @ p.T, 1), (dq, r @ dx.T, r.abs() @ size.T, 3),
                                      (dr, q @ dx + d @ p, q.abs() @ size + d.abs() @ p, 3)):
        err = (got - want).abs() - HALF[BF16] * (roundings * mag + want.abs()) - 1e-30
        assert torch.isfinite(got).all() and float(err.max()) <= 0


# ------------------------------------------------------------------------------------------------ streams and graphs
@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_captured_training_step(sc, dtype):
    """Forward and gradients in a graph, replayed on changed inputs beside eager calls."""
    q, r, v = cuda(*inputs(dtype, 2, 64, (20, 20), 45, 64, seed=90))
    d_out = rand(91, (2, 64, 45), dtype, unit=False).cuda()
    mask = silhouette(92, 2, 20, 20).cuda()
    opts = dict(scale=15.0, cap=6.0, mask=mask)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        gradients(sc, q, r, v, d_out, None, **opts)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, grads = gradients(sc, q, r, v, d_out, None, **opts)
    for seed in range(4):
        fresh = cuda(*inputs(dtype, 2, 64, (20, 20), 45, 64, seed=100 + seed))
        for a, b in zip((q, r, v), fresh):
            a.copy_(b)
        mask.copy_(silhouette(110 + seed, 2, 20, 20))
        want = gradients(sc, q, r, v, d_out, None, **opts)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and all(torch.equal(a, b) for a, b in zip(grads, want[1]))


@gpu
def test_two_streams_share_nothing(sc):
    sets = [cuda(*inputs(F32, 1, 64, (24, 24), 9, 0, seed=120 + 10 * i)) for i in range(2)]
    want = [sc.soft_match(q, r, scale=10.0) for q, r, _ in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(10):
        for i, (q, r, _) in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                got[i].append(sc.soft_match(q, r, scale=10.0))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


# ------------------------------------------------------------------------------------------------ store
def scales(largest, top):
    """A scale is the largest magnitude times the float32 number next to 1 / top, rounded to float32."""
    return largest.astype(np.float32) * (np.float32(1) / np.float32(top))


def quantised(x, kind):
    """(n,C,m) float64 -> values, scales in 64 bits from float32 scales."""
    top = 127.0 if kind == "int8" else 448.0
    s = scales(np.abs(x).max(1), top).astype(np.float64)
    y = np.divide(x, s[:, None], out=np.zeros_like(x), where=s[:, None] > 0).clip(-top, top)
    if kind == "int8":
        return np.rint(y) * s[:, None], s
    e = np.maximum(np.frexp(y)[1] - 1, -6)
    step = np.ldexp(1.0, e - 3)
    return np.rint(y / step) * step * s[:, None], s


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("n, c, size", [(1, 1, (1, 1)), (5, 128, (28, 28)), (3, 37, (9, 15)), (2, 256, (1, 65))])
def test_store_round_trip(sc, dtype, kind, n, c, size):
    x = rand(n, (n, c) + size, F32, unit=False)
    x *= torch.exp(3 * torch.randn((n, 1) + size, generator=torch.Generator().manual_seed(1)))
    x[0, :, 0, 0] = 0
    x = x.to(dtype)
    store = sc.TemplateStore(n + 2, c, size, kind)
    order = torch.randperm(n + 2, generator=torch.Generator().manual_seed(2))[:n].to(torch.int32)
    store.write(order.cuda(), x.cuda())
    want, s = quantised(flat(x), kind)
    assert np.array_equal(host(store.scales[order.long().cuda()]), s)
    got = store.read(order.cuda())
    assert got.shape == x.shape and np.array_equal(flat(got).astype(np.float32), want.astype(np.float32))
    half = store.read(order.cuda(), dtype=BF16)
    assert torch.equal(half, got.to(BF16))
    assert (store.read_mask(order.cuda()) == 1).all()
    unwritten = [i for i in range(n + 2) if i not in order.tolist()]
    assert (store.read(unwritten) == 0).all() and (store.read_mask(unwritten) == 0).all()
    # reading back what was read and writing it again changes no code
    codes = store.codes.clone()
    store.write(order, got)
    assert torch.equal(store.codes.view(torch.uint8), codes.view(torch.uint8))


@gpu
@pytest.mark.parametrize("kind", ["int8", "fp8"])
def test_store_borders(sc, kind):
    """Values that lie on, and a float32 step beside, the border between two codes; the tiniest and largest scales."""
    top = 127.0 if kind == "int8" else 448.0
    levels = np.arange(-126.5, 127, 1.0) if kind == "int8" else np.concatenate([(np.arange(8, 16) + 0.5) * 2.0 ** e for e in range(-9, 5)] + [(np.arange(8) + 0.5) * 2.0 ** -9])
    levels = levels[np.abs(levels) < top]
    for largest in (top, 0.37, 1e-25, 3e30):
        largest = np.full((3, 1), largest, np.float32)
        base = (levels * scales(largest[0], top)).astype(np.float32)
        x = np.stack([base, np.nextafter(base, np.float32(np.inf)), np.nextafter(base, -np.float32(np.inf))])
        x = np.concatenate([x, largest], 1)[:, :, None]                                              # (3, C, 1)
        store = sc.TemplateStore(3, x.shape[1], (1, 1), kind)
        store.write([0, 1, 2], x[..., None])
        want, _ = quantised(x.astype(np.float64), kind)
        got = host(store.read([0, 1, 2])).reshape(want.shape)
        assert np.array_equal(got.astype(np.float32), want.astype(np.float32)), largest[0, 0]


@gpu
def test_store_bad_cells_repeats_and_absent_views(sc):
    x = rand(1, (4, 16, 3, 5), F32, unit=False)
    x[1, 3, 1, 2] = float("nan")
    x[1, 0, 2, 4] = float("inf")
    take = silhouette(2, 4, 3, 5)
    take[1] = True
    store = sc.TemplateStore(6, 16, (3, 5))
    untouched = store.codes.clone()
    # view 2 twice: its last entry stays; indices outside the store are skipped (device indices)
    store.write(torch.tensor([2, 0, 2, -1], device="cuda"), x.cuda(), mask=take.cuda())
    assert torch.equal(store.codes[[1, 3, 4, 5]], untouched[[1, 3, 4, 5]])
    assert np.array_equal(flat(store.read([2]))[0].astype(np.float32), quantised(flat(x[2:3]), "int8")[0][0].astype(np.float32))
    mask = store.read_mask([2, 0])
    assert torch.equal(mask[0].cpu().bool(), take[2])
    good = torch.ones((3, 5), dtype=torch.bool)
    good[1, 2] = good[2, 4] = False
    assert torch.equal(mask[1].cpu().bool(), good) and torch.isfinite(store.read([0])).all()
    far = torch.tensor([2 ** 32 + 2, 77, -5, 2], device="cuda")
    got = store.read(far)
    assert (got[:3] == 0).all() and torch.equal(got[3], store.read([2])[0])
    assert (store.read_mask(far)[:3] == 0).all()
    before = store.codes.clone()
    store.write(far[:3], x[:3].cuda())
    assert torch.equal(store.codes, before)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("b, v, n, c, heads, size, cap", [(1, 1, 1, 128, 1, (28, 28), 0.0), (3, 3, 10, 64, 2, (9, 13), 6.0),
                                                         (2, 5, 70, 100, 1, (7, 9), 0.0), (1, 2, 200, 256, 1, (8, 8), 5.0)])
def test_store_match(sc, dtype, kind, b, v, n, c, heads, size, cap):
    store = sc.TemplateStore(8, c, size, kind)
    feats = rand(3, (8, c) + size, F32)
    mask = silhouette(4, 8, *size)
    store.write(range(7), feats[:7], mask=mask[:7])
    g = torch.Generator().manual_seed(5)
    views = torch.stack([torch.randperm(8, generator=g)[:v] for _ in range(b)])
    if v > 1:
        views[0, 1] = -1                                 # one absent view
        views[-1, 0] = 7                                 # one not yet written
    q = rand(6, (b, c, n), dtype)
    out, lse = store.soft_match(q.cuda(), views.cuda(), heads=heads, scale=20.0, cap=cap, return_lse=True)
    at = views.clamp_min(0).reshape(-1).tolist()
    values = flat(store.read(at)).reshape(b, v, c, -1).transpose(0, 2, 1, 3).reshape(b, c, -1)
    masks = host(store.read_mask(at)).reshape(b, v, -1) * (views >= 0).numpy()[:, :, None]
    want = oracle(flat(q), values, values, heads, 20.0, cap, mask=masks.reshape(b, -1))
    near(out, want[0], want[2], dtype, 1)
    near_lse(lse, want[1])
    assert torch.equal(store.soft_match(q.cuda(), views.tolist(), heads=heads, scale=20.0, cap=cap), out)


@gpu
def test_store_match_options(sc):
    size = (6, 7)
    store = sc.TemplateStore(4, 32, size)
    store.write(range(4), rand(7, (4, 32) + size, F32))
    q = rand(8, (2, 32) + size, F32)
    views = [[0, 3], [2, 2]]
    out = store.soft_match(q.cuda(), views, scale=10.0, falloff=0.1, num_query=[42, 5])
    values = flat(store.read([0, 3, 2, 2])).reshape(2, 2, 32, 42).transpose(0, 2, 1, 3)
    outs = []
    for i in range(2):
        # the grid repeats for every view: one oracle item per layout of cells
        m = values[i].reshape(1, 32, 84)
        x = 10.0 * host(q)[i].reshape(32, 42).T @ m[0]
        cell = np.stack([np.arange(84) % 42 % 7, np.arange(84) % 42 // 7], 1)
        place = np.stack([np.arange(42) % 7, np.arange(42) // 7], 1)
        z = x - 0.1 * ((place[:, None] - cell[None]) ** 2).sum(2)
        p = np.exp(z - z.max(1, keepdims=True))
        outs.append(m[0] @ (p / p.sum(1, keepdims=True)).T)
    outs[1][:, 5:] = 0
    assert np.abs(flat(out) - np.stack(outs)).max() <= 2e-5
    none = store.soft_match(q.cuda(), torch.full((2, 3), -1), return_lse=True)
    assert (none[0] == 0).all() and torch.isneginf(none[1]).all()
    none = store.soft_match(q.cuda(), torch.empty((2, 0), dtype=torch.int64), return_lse=True)
    assert (none[0] == 0).all() and torch.isneginf(none[1]).all()


@gpu
def test_store_beyond_32_bit_offsets(sc):
    """Views whose codes lie more than 2^31 bytes into the store."""
    n, c, size = 2100, 256, (64, 64)                     # 2.2 GB of codes
    store = sc.TemplateStore(n, c, size)
    x = rand(1, (2, c) + size, F32)
    store.write([n - 1, 0], x)
    got = store.read([n - 1, 0])
    want, _ = quantised(flat(x), "int8")
    assert np.array_equal(flat(got).astype(np.float32), want.astype(np.float32))
    q = rand(2, (1, c, 4), F32)
    out = store.soft_match(q.cuda(), [[n - 1]], scale=20.0)
    ref = oracle(flat(q), want[:1], want[:1], 1, 20.0)
    near(out, ref[0], ref[2], F32, 1)


@gpu
@pytest.mark.parametrize("kind", ["int8", "fp8"])
def test_templates_from_poses_to_matches(sc, kind):
    """As a matching step uses them: views written once, the nearest views of a batch looked up, matched softly straight from
    the codes, and read back for the hard match."""
    from pose_estimation_amd import correspondence
    poses = np.array([[az, 10.0, 0.0] for az in range(0, 360, 45)])
    feats = correspondence.l2norm(rand(11, (8, 128, 14, 14), F32).cuda())
    object_ = silhouette(12, 8, 14, 14, share=0.7).cuda()
    store = sc.TemplateStore(8, 128, (14, 14), kind)
    store.write(range(8), feats, mask=object_)
    asked = np.array([[[46.0, 8.0, 0.0], [359.0, 12.0, 3.0]], [[180.0, 10.0, 1.0], [91.0, 10.0, 0.0]]])
    views = correspondence.nearest_view(asked.reshape(-1, 3), poses).reshape(2, 2)
    assert views.tolist() == [[1, 0], [4, 2]]
    cells = torch.stack([torch.nonzero(object_[v].flatten())[:9, 0] for v in views[:, 0]])
    q = feats[torch.as_tensor(views[:, 0]).cuda()].flatten(2).gather(2, cells[:, None].expand(2, 128, 9))
    out, lse = store.soft_match(q, views, scale=60.0, return_lse=True)
    back = store.read(views[:, 0])
    dist, ind = correspondence.dense_nn(q, back, 1, index_base=0)
    assert torch.equal(ind[:, 0].long(), cells)
    # other cells lie a cosine of more than 0.5 lower: weights below exp(-30); codes are 2^-4 of themselves off at most
    hit = back.flatten(2).gather(2, cells[:, None].expand(2, 128, 9))
    assert torch.allclose(out, hit, rtol=1e-4, atol=1e-5)
    assert torch.allclose(lse[:, 0], 60.0 * (q * hit).sum(1), rtol=1e-5)
    # the same against the maps that the codes stand for
    maps = store.read(views.reshape(-1)).view(2, 2, 128, -1).transpose(1, 2).flatten(2)
    masks = store.read_mask(views.reshape(-1)).view(2, 1, -1)
    same = sc.soft_match(q, maps, scale=60.0, mask=masks)
    assert torch.allclose(out, same, rtol=1e-4, atol=1e-5)


# ------------------------------------------------------------------------------------------------ every form of the kernels
# More than 64 queries and cells take workgroups of four waves, with a form of their own for plain scores, for caps up to 32
# (bfloat16), for a falloff on a grid whose width is a multiple of 8 cells, and for the rest.
SCORES = {
    "plain": dict(scale=15.0),
    "negative scale": dict(scale=-15.0),
    "no scale": dict(scale=0.0),
    "cap": dict(scale=25.0, cap=6.0),
    "large cap": dict(scale=25.0, cap=40.0),
    "falloff": dict(scale=15.0, falloff=0.04),
    "rising falloff": dict(scale=-15.0, falloff=-0.02),
    "falloff alone": dict(scale=0.0, falloff=0.04),
    "cap and falloff": dict(scale=25.0, cap=6.0, falloff=0.04),
}
FORMS = [  # channels, heads, value channels, queries (0: the grid)
    (32, 1, 0, 0),
    (128, 2, 64, 150),
    (128, 1, 0, 150),
    (100, 1, 128, 0),
    (256, 1, 0, 0),
    (200, 1, 256, 150),
]


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("scores", SCORES)
def test_forms(sc, dtype, form, scores):
    """Forward and gradients of an item of whole and one of partly masked, partly real rows."""
    c, heads, cv, n = form
    grid, nq = (15, 24), form[3] or 360
    q, r, v = inputs(dtype, 2, c, grid, n, cv, seed=130)
    opts = dict(SCORES[scores])
    fall = xy = None
    if "falloff" in opts:
        fall = opts["falloff"] = torch.full((heads,), opts["falloff"])
        if n:
            xy = opts["query_xy"] = torch.rand((2, n, 2), generator=torch.Generator().manual_seed(3)) * torch.tensor([23.0, 14.0])
    mask = torch.ones((2,) + grid, dtype=torch.bool)
    mask[1] = silhouette(131, 1, *grid)[0]
    count = torch.tensor([nq, nq - 47])
    d_out, d_lse = rand(132, (2, cv or c) + tuple(q.shape[2:]), dtype, unit=False), rand(133, (2, heads, nq), F32, unit=False)
    out, got = gradients(sc, *cuda(q, r, v, d_out, d_lse), heads=heads, mask=mask.cuda(), num_query=count, **opts)
    want = oracle(flat(q), flat(r), flat(r if v is None else v), heads, opts["scale"], opts.get("cap", 0.0),
                  None if fall is None else host(fall), None if xy is None else host(xy), grid[1], mask.numpy(), count.numpy(),
                  flat(d_out), host(d_lse))
    near(out, want[0], want[2], dtype, 1)
    check_gradients(got, want, dtype, v is None)


@gpu
@pytest.mark.parametrize("grid", [(12, 16), (12, 15)])
@pytest.mark.parametrize("falloff", [2.0, 50.0])
def test_steep_falloff(sc, falloff, grid):
    """Distances as exact as float32 has them: queries between cells, whose nearest ones weigh alike."""
    q, r, v = inputs(F32, 1, 16, grid, 100, 8, seed=140)
    xy = torch.rand((1, 100, 2), generator=torch.Generator().manual_seed(141)) * torch.tensor([grid[1] - 1.0, grid[0] - 1.0])
    out, lse = sc.soft_match(*cuda(q, r, v), scale=4.0, falloff=falloff, query_xy=xy, return_lse=True)
    want = oracle(flat(q), flat(r), flat(v), 1, 4.0, 0.0, [falloff], host(xy), grid[1])
    # scores of the cells that count: up to falloff / 2 + 4 = 29, below the 60 of the tolerance's count
    near(out, want[0], want[2], F32, 1)
    near_lse(lse, want[1])


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n, grid, cv", [(100, (64, 80), 0), (70, (72, 70), 32), (900, (30, 34), 0), (3, (100, 100), 0), (64, (50, 41), 8)])
def test_many_parts(sc, dtype, n, grid, cv):
    """Few workgroups: the cells are split over many, whose parts are joined."""
    q, r, v = inputs(dtype, 1, 32, grid, n, cv, seed=150)
    mask = silhouette(151, 1, *grid)
    mask[0, : grid[0] // 2] = False                      # parts without a cell
    d_out, d_lse = rand(152, (1, cv or 32, n), dtype, unit=False), rand(153, (1, 1, n), F32, unit=False)
    out, got = gradients(sc, *cuda(q, r, v, d_out, d_lse), scale=20.0, mask=mask[:, None].cuda())
    want = oracle(flat(q), flat(r), flat(r if v is None else v), 1, 20.0, mask=mask.numpy(), d_out=flat(d_out), d_lse=host(d_lse))
    near(out, want[0], want[2], dtype, 1)
    check_gradients(got, want, dtype, v is None)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_one_cell_far_above_the_rest(sc, dtype):
    """The largest score rises late, in steps beyond and within what the sums are kept for, in each tile of 64 cells."""
    n, m, c = 130, 640, 32
    q, r = rand(160, (1, c, n), dtype), rand(161, (1, c, m), dtype) * 0.01
    for k, size in enumerate((0.05, 0.1, 0.3, 0.35, 0.9, 1.0)):
        at = 5 + 101 * k
        r[0, :, at] = q[0, :, 17 * k] * size
    out, lse = sc.soft_match(q.cuda(), r.cuda(), scale=80.0, return_lse=True)
    want = oracle(flat(q), flat(r), flat(r), 1, 80.0)
    near(out, want[0], want[2], dtype, 1)
    # scores up to 80: 80 2^-24 of a weight each, in the tolerance of near_lse
    near_lse(lse, want[1])


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("c, heads, size, n", [(128, 1, (10, 16), 0), (128, 1, (9, 13), 100), (256, 1, (6, 8), 100), (64, 2, (7, 8), 20)])
def test_store_match_falloff(sc, dtype, kind, c, heads, size, n):
    """The grid's distances in every view, per head; the same as soft_match over the views side by side."""
    h, w = size
    store = sc.TemplateStore(5, c, size, kind)
    store.write(range(5), rand(170, (5, c) + size, F32), mask=silhouette(171, 5, h, w))
    views = [[4, 0, 2], [1, 1, -1]]
    nq = n or h * w
    q = rand(172, (2, c, n) if n else (2, c, h, w), dtype)
    xy = torch.rand((2, n, 2), generator=torch.Generator().manual_seed(173)) * torch.tensor([w - 1.0, h - 1.0]) if n else None
    fall = [0.03 * (i + 1) for i in range(heads)]
    out, lse = store.soft_match(q.cuda(), views, heads=heads, scale=18.0, falloff=fall, query_xy=xy, num_query=[nq, nq - 7],
                                return_lse=True)
    ids = np.maximum(np.array(views).reshape(-1), 0)
    values = flat(store.read(ids)).reshape(2, 3, c, -1).transpose(0, 2, 1, 3).reshape(2, c, -1)
    masks = (host(store.read_mask(ids)).reshape(2, 3, -1) * (np.array(views) >= 0)[:, :, None]).reshape(2, -1)
    # the oracle's grid is one map: per view, joined by the log-sums
    want, mag, want_lse = 0, 0, None
    parts = [oracle(flat(q), values[:, :, i * h * w:(i + 1) * h * w], values[:, :, i * h * w:(i + 1) * h * w], heads, 18.0, 0.0, fall,
                    None if xy is None else host(xy), w, masks[:, i * h * w:(i + 1) * h * w], [nq, nq - 7]) for i in range(3)]
    want_lse = np.logaddexp.reduce([p[1] for p in parts])
    for p in parts:
        share = np.where(np.isneginf(p[1]), 0, np.exp(p[1] - np.where(np.isneginf(want_lse), 0, want_lse)))
        share = np.repeat(share, c // heads, 1)
        want, mag = want + share * p[0], mag + share * p[2]
    near(out, want, mag, dtype, 1)
    near_lse(lse, want_lse)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("n, c, heads, size, views", [(1, 128, 1, (1, 1), 2), (8, 128, 1, (1, 7), 1), (7, 40, 2, (1, 9), 3), (1, 256, 1, (23, 29), 4),
                                                      (8, 256, 2, (40, 41), 3), (9, 64, 1, (2, 3), 2), (3, 5, 1, (64, 64), 30), (1, 12, 3, (130, 130), 5)])
@pytest.mark.parametrize("cap, falloff", [(0.0, None), (6.0, None), (9.0, 0.02)])
def test_store_match_few_queries(sc, dtype, kind, n, c, heads, size, views, cap, falloff):
    """Up to 8 queries, rows of codes that end inside a tile or are shorter than a segment, features of any size."""
    h, w = size
    store = sc.TemplateStore(views, c, size, kind)
    feats = rand(200, (views, c) + size, F32) * torch.exp(torch.randn((views, 1) + size, generator=torch.Generator().manual_seed(201)) * 0.3)
    mask = silhouette(202, views, h, w)
    mask[0, 0, 0] = True
    store.write(range(views), feats, mask=mask)
    q = rand(203, (2, c, n), dtype)
    xy = torch.rand((2, n, 2), generator=torch.Generator().manual_seed(204)) * torch.tensor([w - 1.0, h - 1.0])
    opts = dict(heads=heads, scale=14.0, cap=cap, falloff=falloff, query_xy=xy if falloff else None, num_query=[n, max(n - 2, 1)])
    out, lse = store.soft_match(q.cuda(), [list(range(views))] * 2, return_lse=True, **opts)
    values = np.broadcast_to(flat(store.read(range(views))).transpose(1, 0, 2).reshape(c, -1), (2, c, views * h * w))
    taken = np.broadcast_to(mask.numpy().reshape(-1), (2, views * h * w))
    if falloff:                                          # per view, joined by the log-sums
        parts = [oracle(flat(q), values[:, :, i * h * w:(i + 1) * h * w], values[:, :, i * h * w:(i + 1) * h * w], heads, 14.0, cap,
                        [falloff] * heads, host(xy), w, taken[:, i * h * w:(i + 1) * h * w], opts["num_query"]) for i in range(views)]
        want_lse = np.logaddexp.reduce([p[1] for p in parts])
        share = [np.repeat(np.where(np.isneginf(p[1]), 0, np.exp(p[1] - np.where(np.isneginf(want_lse), 0, want_lse))), c // heads, 1)
                 for p in parts]
        want, mag = sum(s * p[0] for s, p in zip(share, parts)), sum(s * p[2] for s, p in zip(share, parts))
    else:
        want, want_lse, mag = oracle(flat(q), values, values, heads, 14.0, cap, mask=taken, count=opts["num_query"])[:3]
    near(out, want, mag, dtype, 1)
    near_lse(lse, want_lse)


@gpu
def test_store_over_a_part_of_another(sc):
    """Views of a larger tensor, which start anywhere."""
    store = sc.TemplateStore(4, 9, (5, 7))
    store.write(range(4), rand(180, (4, 9, 5, 7), F32))
    part = sc.TemplateStore.from_tensors(store.codes[1:], store.scales[1:], store.mask[1:], (5, 7))
    assert torch.equal(part.read([0, 2]), store.read([1, 3]))
    q = rand(181, (1, 9, 90), F32).cuda()
    assert torch.equal(part.soft_match(q, [[0, 2]], scale=9.0), store.soft_match(q, [[1, 3]], scale=9.0))
    part.write([1], rand(182, (1, 9, 5, 7), F32))
    assert torch.equal(part.read([1]), store.read([2]))


@gpu
def test_captured_store(sc):
    """Write, match and read in a graph, replayed on other views."""
    feats = rand(190, (6, 32, 8, 9), F32).cuda()
    store, twin = sc.TemplateStore(6, 32, (8, 9)), sc.TemplateStore(6, 32, (8, 9))
    views, x, q = torch.zeros(2, dtype=torch.int32, device="cuda"), feats[:2].clone(), rand(191, (1, 32, 70), F32).cuda()

    def step(s):
        s.write(views, x)
        return s.soft_match(q, views[None], scale=15.0), s.read(views), s.read_mask(views)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(store)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(store)
    for i in range(3):
        views.copy_(torch.tensor([5 - i, i]))
        x.copy_(feats[2 * i:2 * i + 2])
        want = step(twin)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n, c", [(0, 32), (9, 32), (0, 256)])
@pytest.mark.parametrize("ratio", [4.0, -4.0, 6.0, -6.0, 8.0, -8.0])
def test_gradients_of_saturated_caps(sc, dtype, n, c, ratio):
    """All cells alike, so that every score lies far in the cap, where 1 - tanh^2 is 1e-3 to 4e-7: its relative error counts.
    It goes by twice that of scale x / cap, a sum of up to 256 terms times 8: 2 x 8 x 8 half steps of 2^-24, 8e-6."""
    grid, cap = (12, 16), 7.0
    q, r, v = inputs(dtype, 2, c, grid, n, 24, seed=220)
    q, r = ((0.1 * x.float() + rand(223, (1, c) + (1,) * (x.dim() - 2), F32)).to(dtype) for x in (q, r))
    d_out = rand(224, (2, 24) + tuple(q.shape[2:]), dtype, unit=False)
    _, got = gradients(sc, *cuda(q, r, v, d_out), None, scale=ratio * cap, cap=cap)
    want = oracle(flat(q), flat(r), flat(v), 1, ratio * cap, cap, d_out=flat(d_out))
    check_gradients(got, want, dtype, False)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n, c", [(0, 48), (5, 48), (0, 256)])
@pytest.mark.parametrize("cap", [33.0, 64.0, 1e3, 1e5, 1e7])
@pytest.mark.parametrize("falloff", [None, 0.03])
def test_caps_that_hardly_bend(sc, dtype, n, c, cap, falloff):
    """A cap far above the scores leaves them as they are: its tanh counts with the cap's size."""
    grid = (15, 16)
    q, r, v = inputs(dtype, 2, c, grid, n, 40, seed=230)
    nq = n or 240
    xy = torch.rand((2, n, 2), generator=torch.Generator().manual_seed(231)) * 14 if n and falloff else None
    d_out, d_lse = rand(232, (2, 40) + tuple(q.shape[2:]), dtype, unit=False), rand(233, (2, 1, nq), F32, unit=False)
    opts = dict(scale=30.0, cap=cap, falloff=falloff, query_xy=xy)
    _, lse = sc.soft_match(*cuda(q, r, v), return_lse=True, **opts)
    out, got = gradients(sc, *cuda(q, r, v, d_out, d_lse), **opts)
    want = oracle(flat(q), flat(r), flat(v), 1, 30.0, cap, None if falloff is None else [falloff], None if xy is None else host(xy), 16,
                  d_out=flat(d_out), d_lse=host(d_lse))
    near(out, want[0], want[2], dtype, 1)
    near_lse(lse, want[1])
    check_gradients(got, want, dtype, False)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cap", [0.0, 6.0])
@pytest.mark.parametrize("grid", [(40, 48), (31, 45)])
@pytest.mark.parametrize("falloff", [1.0, 40.0, 1e3, 3e4])
def test_steep_falloff_on_the_grid(sc, dtype, falloff, grid, cap):
    """Queries on cells: the distance of the cell that counts is 0, so scores are as exact as without a falloff, however far
    those of the cells before it lie below."""
    q, r, v = inputs(dtype, 1, 32, grid, 0, 8, seed=240)
    n = grid[0] * grid[1]
    d_out, d_lse = rand(241, (1, 8) + grid, dtype, unit=False), rand(242, (1, 1, n), F32, unit=False)
    opts = dict(scale=12.0, falloff=falloff, cap=cap)
    _, lse = sc.soft_match(*cuda(q, r, v), return_lse=True, **opts)
    out, got = gradients(sc, *cuda(q, r, v, d_out, d_lse), **opts)
    want = oracle(flat(q), flat(r), flat(v), 1, 12.0, cap, [falloff], None, grid[1], d_out=flat(d_out), d_lse=host(d_lse))
    near(out, want[0], want[2], dtype, 1)
    near_lse(lse, want[1])
    check_gradients(got, want, dtype, False)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("grid", [(40, 48), (31, 45)])
@pytest.mark.parametrize("n", [7, 50, 200])
@pytest.mark.parametrize("falloff", [1.0, 1e3, 3e4])
def test_store_match_steep_falloff(sc, dtype, falloff, n, grid):
    """The same against a stored view: queries on whole cells of the grid."""
    store = sc.TemplateStore(1, 32, grid)
    store.write([0], rand(250, (1, 32) + grid, F32))
    q = rand(251, (1, 32, n), dtype)
    g = torch.Generator().manual_seed(252)
    xy = torch.stack([torch.randint(grid[1], (1, n), generator=g), torch.randint(grid[0], (1, n), generator=g)], 2).float()
    out, lse = store.soft_match(q.cuda(), [[0]], scale=12.0, falloff=falloff, query_xy=xy, return_lse=True)
    values = flat(store.read([0]))
    want = oracle(flat(q), values, values, 1, 12.0, 0.0, [falloff], host(xy), grid[1])
    near(out, want[0], want[2], dtype, 1)
    near_lse(lse, want[1])


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("stored", [False, True])
@pytest.mark.parametrize("grid", [(40, 48), (31, 45)])
@pytest.mark.parametrize("n, items", [(0, 48), (50, 1100)])
@pytest.mark.parametrize("falloff", [40.0, 3e4, 3e7])
def test_scores_that_rise_late(sc, dtype, stored, grid, n, items, falloff):
    """Workgroups that walk the whole map, over cells whose scores lie up to 1e11 below those that count.  All items are alike."""
    q, r, _ = inputs(dtype, 1, 32, grid, n, 0, seed=260)
    g = torch.Generator().manual_seed(261)
    xy = torch.stack([torch.randint(grid[1], (1, n), generator=g), torch.randint(grid[0], (1, n), generator=g)], 2).float() if n else None
    opts = dict(scale=12.0, falloff=falloff, query_xy=xy.expand(items, -1, -1).contiguous() if n else None, return_lse=True)
    many = q.cuda().expand((items,) + tuple(q.shape[1:])).contiguous()
    if stored:
        store = sc.TemplateStore(1, 32, grid)
        store.write([0], r)
        out, lse = store.soft_match(many, [[0]] * items, **opts)
        r = store.read([0])
    else:
        out, lse = sc.soft_match(many, r.cuda().expand((items,) + tuple(r.shape[1:])), **opts)
    want = oracle(flat(q), flat(r), flat(r), 1, 12.0, 0.0, [falloff], host(xy) if n else None, grid[1])
    near(out[:1], want[0], want[2], dtype, 1)
    near_lse(lse[:1], want[1])
    assert (out == out[:1]).all() and (lse == lse[:1]).all()


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [5, 100])
@pytest.mark.parametrize("cap", [0.0, 1e9])
@pytest.mark.parametrize("scale", [1e6, -1e8, 1e9, -1e12, 1e20])
def test_scores_of_any_size(sc, dtype, n, cap, scale):
    """Scores whose float32 steps are wider than the exponents of the softmax: the largest one takes all."""
    q, r, v = inputs(dtype, 1, 32, (20, 20), n, 16, seed=270)
    mask = silhouette(271, 1, 20, 20)
    mask[0, :5] = False                                  # tiles without a cell first
    out, lse = sc.soft_match(*cuda(q, r, v), scale=scale, cap=cap, mask=mask.cuda(), return_lse=True)
    want = oracle(flat(q), flat(r), flat(v), 1, scale, cap, mask=mask.numpy())
    # a score is a sum of 32 rounded terms, and rounded as it is stored: 40 2^-24 of the largest at most
    assert np.isfinite(host(out)).all() and np.abs(host(lse) / want[1] - 1).max() <= 40 * 2.0 ** -24
    x = scale * flat(q)[0].T @ flat(r)[0][:, mask.numpy().reshape(-1)]
    z = np.sort(cap * np.tanh(x / cap) if cap else x, 1)
    clear = z[:, -1] - z[:, -2] > 100 * 2.0 ** -24 * np.abs(z).max() + 100
    assert clear.any() or cap
    # the one weight is 2^x with |x| <= 1, not 1, and is divided by itself: w v, 1 / l and their product are rounded as any weight's
    # are, so that the bound is near's (float32: 3 half steps and what the planes' product leaves out, 8 half steps, below 2e-5)
    slack = 2e-5 if dtype == F32 else HALF[dtype]
    err = np.abs(flat(out) - want[0])[0][:, clear]
    assert (err <= (slack + HALF[dtype]) * np.abs(want[0][0][:, clear])).all()
    # no average leaves the values' range
    assert np.abs(host(out)).max() <= np.abs(host(v)).max() * (1 + slack + HALF[dtype])


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [5, 100])
@pytest.mark.parametrize("opts", [dict(), dict(cap=1e9), dict(falloff=0.05), dict(cap=1e13, falloff=0.05)])
@pytest.mark.parametrize("scale", [1e9, -1e12, 1e20])
def test_gradients_of_scores_of_any_size(sc, dtype, n, opts, scale):
    """A weight formed from a log-sum that is wider rounded than an exponent is still a weight: at most 1."""
    q, r, v = inputs(dtype, 1, 32, (20, 24), n, 16, seed=280)
    if "falloff" in opts:
        opts = opts | dict(query_xy=torch.rand((1, n, 2), generator=torch.Generator().manual_seed(281)) * 19)
    d_out = rand(282, (1, 16, n), dtype, unit=False)
    out, got = gradients(sc, *cuda(q, r, v, d_out), None, scale=scale, **opts)
    assert np.isfinite(host(out)).all() and all(np.isfinite(host(g)).all() for g in got)
    most = np.abs(host(d_out)).sum(2)[:, :, None, None]
    assert (np.abs(host(got[2])) <= most * (1 + n * HALF[dtype])).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.uint16, torch.int16, torch.uint32, torch.int32, torch.int64])
def test_counts_of_every_type(sc, dtype):
    """A count above every query map means all of it, also one that int32 does not hold."""
    q, r, _ = inputs(F32, 2, 16, (5, 6), 40, seed=290)
    most = min(torch.iinfo(dtype).max, 2 ** 63 - 1)
    count = torch.from_numpy(np.array([most, 7], dtype=str(dtype).split(".")[1]))
    want = sc.soft_match(*cuda(q, r), num_query=[40, 7])
    for x in (count, count.cuda()):
        assert torch.equal(sc.soft_match(*cuda(q, r), num_query=x), want)


# ------------------------------------------------------------------------------------------------ refusals (no GPU)
def test_refusals(sc):
    q, r = torch.zeros((2, 8, 4, 4)), torch.zeros((2, 8, 5, 6))
    bad = [
        (dict(query=torch.zeros((2, 8))), "must be"),
        (dict(ref=torch.zeros((1, 8, 5, 6))), "share batch and channels"),
        (dict(ref=torch.zeros((2, 7, 5, 6))), "share batch and channels"),
        (dict(ref=torch.zeros((2, 8, 0, 6))), "no cells"),
        (dict(ref=r.to(BF16)), "dtype"),
        (dict(query=q.half(), ref=r.half()), "float32 or bfloat16"),
        (dict(query=q.double(), ref=r.double()), "float32 or bfloat16"),
        (dict(value=torch.zeros((2, 4, 5, 5))), "batch and cells"),
        (dict(value=torch.zeros((1, 4, 5, 6))), "batch and cells"),
        (dict(value=torch.zeros((2, 4, 5, 6), dtype=BF16)), "dtype"),
        (dict(heads=3), "heads"),
        (dict(heads=0), "heads"),
        (dict(heads=8, value=torch.zeros((2, 4, 5, 6))), "heads"),
        (dict(query=torch.zeros((2, 257, 3)), ref=torch.zeros((2, 257, 3))), "at most 256"),
        (dict(scale=math.inf), "scale"),
        (dict(cap=-1.0), "cap"),
        (dict(cap=math.nan), "cap"),
        (dict(falloff=0.1), "do not lie on the reference grid"),
        (dict(ref=torch.zeros((2, 8, 30)), falloff=0.1), "on its grid"),
        (dict(falloff=[0.1, 0.2], query_xy=torch.zeros((2, 16, 2))), "per head"),
        (dict(falloff=0.1, query_xy=torch.zeros((2, 15, 2))), "query_xy"),
        (dict(mask=torch.ones((2, 5, 5))), "mask"),
        (dict(mask=torch.ones((1, 5, 6))), "mask"),
        (dict(num_query=[1, 2, 3]), "one count per"),
        (dict(num_query=[1.5, 2.0]), "integers"),
        (dict(num_query=torch.ones(2)), "integers"),
        (dict(mask=[[True] * 6] * 5), "mask"),
        (dict(mask=torch.ones((2, 6, 5))), "mask"),
        (dict(query=q[..., :3, :3], falloff=math.nan, query_xy=torch.zeros((2, 9, 2))), "finite"),
        (dict(falloff=[math.inf], query_xy=torch.zeros((2, 16, 2))), "finite"),
        (dict(query=[[1.0, 2.0]]), "must be"),
        (dict(query=q.clone().requires_grad_(), ref=r.numpy()), "must be tensors"),
    ]
    for args, match in bad:
        call = dict(query=q, ref=r) | args
        with pytest.raises(ValueError, match=match):
            sc.soft_match(call.pop("query"), call.pop("ref"), call.pop("value", None), **call)


def test_counts_of_other_types_are_refused(sc):
    q, r = torch.zeros((2, 8, 4, 4)), torch.zeros((2, 8, 5, 6))
    for dtype in (torch.bool, torch.complex64, torch.uint64, torch.float16):
        with pytest.raises(ValueError, match="num_query must hold integers"):
            sc.soft_match(q, r, num_query=torch.ones(2).to(dtype))
    with pytest.raises(ValueError, match="num_query must hold integers"):
        sc.soft_match(q, r, num_query=[True, False])


def test_numbers_that_float32_does_not_hold_are_refused(sc):
    from pose_estimation_amd import _abi
    q, r = torch.zeros((2, 8, 5, 6)), torch.zeros((2, 8, 5, 6))
    for args, match in [(dict(cap=1e-50), "too small"), (dict(cap=1e-31), "too small"), (dict(cap=1e-5, scale=-1e26), "too small"),
                        (dict(falloff=1e39), "finite in float32"), (dict(falloff=[-1e38]), "finite in float32")]:
        with pytest.raises(ValueError, match=match):
            sc.soft_match(q, r, **args)
    for cap, scale in ((1e-31, 1.0), (1e-5, -1e26)):
        assert _abi.lib.ispa_soft_match(1, 1, None, 0, 1, 1, 64, 64, 10, 100, 10, scale, cap, None, None, None, None, 1, None, None, None, 0,
                                        None) == -1 and b"too small" in _abi.lib.ispa_last_error()


def test_learned_scale_and_cap_are_refused(sc):
    q, r = torch.zeros((2, 8, 4, 4)), torch.zeros((2, 8, 5, 6))
    learned = torch.tensor(3.0, requires_grad=True)
    for x in (q, q.clone().requires_grad_()):
        for name in ("scale", "cap"):
            with pytest.raises(ValueError, match=f"no gradient flows to {name}"):
                sc.soft_match(x, r, **{name: learned})
    # where none is asked for they pass for the numbers they hold: on to the next check
    with torch.no_grad(), pytest.raises(ValueError, match="do not lie on the reference grid"):
        sc.soft_match(q, r, scale=learned, cap=learned, falloff=0.1)
    with pytest.raises(ValueError, match="scale must be finite"):
        sc.soft_match(q, r, scale=(learned / 0).detach())


def test_forward_mode_is_refused(sc):
    from torch.autograd import forward_ad
    q, r, v = torch.zeros((2, 8, 4, 4)), torch.zeros((2, 8, 5, 6)), torch.zeros((2, 4, 5, 6))
    with forward_ad.dual_level():
        dual = [forward_ad.make_dual(x, torch.ones_like(x)) for x in (q, r, v)]
        for i in range(3):
            with pytest.raises(ValueError, match="forward-mode"):
                sc.soft_match(*(dual[j] if j == i else x for j, x in enumerate((q, r, v))))
        with pytest.raises(ValueError, match="forward-mode"):
            sc.soft_match(q, r, scale=forward_ad.make_dual(torch.tensor(2.0), torch.tensor(1.0)))
        with pytest.raises(ValueError, match="heads"):   # a level alone changes nothing
            sc.soft_match(q, r, v, heads=3)
        with pytest.raises(ValueError, match="do not lie on the reference grid"):
            sc.soft_match(q, r, v, falloff=0.1)
    with pytest.raises(ValueError, match="forward-mode"):
        torch.func.jvp(lambda x: sc.soft_match(x, r), (q,), (q,))


def test_store_refusals(sc):
    with pytest.raises(ValueError, match="kind"):
        sc.TemplateStore(1, 8, (4, 4), "int4")
    with pytest.raises(ValueError, match="views of"):
        sc.TemplateStore(0, 8, (4, 4))
    codes = torch.zeros((3, 8, 16), dtype=torch.int8)
    flat_, byte = torch.zeros((3, 16)), torch.zeros((3, 16), dtype=torch.uint8)
    for args, match in [((codes.float(), flat_, byte, (4, 4)), "int8 or float8"), ((codes, flat_, byte, (4, 5)), "no \\(4, 5\\) maps"),
                        ((codes, flat_.double(), byte, (4, 4)), "scales"), ((codes, flat_, byte[:2], (4, 4)), "mask"),
                        ((codes, flat_, byte, (4, 4)), "on one GPU")]:
        with pytest.raises(ValueError, match=match):
            sc.TemplateStore.from_tensors(*args)
    store = sc.TemplateStore.__new__(sc.TemplateStore)
    store._set("int8", 3, 8, (4, 4))
    x = torch.zeros((2, 8, 4, 4))
    for views, error, match in [([0, 3], IndexError, "outside"), ([-2, 0], IndexError, "outside"), ([0.5, 1.0], ValueError, "integers"),
                                ([[0], [1]], ValueError, "1 dimension")]:
        with pytest.raises(error, match=match):
            store.write(views, x)
        with pytest.raises(error, match=match):
            store.read(views)
    with pytest.raises(ValueError, match="features must be"):
        store.write([0], x)
    with pytest.raises(ValueError, match="mask must be"):
        store.write([0, 1], x, mask=torch.ones((2, 4, 3)))
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        store.write([0, 1], x.half())
    with pytest.raises(ValueError, match="dtype"):
        store.read([0], dtype=torch.float16)
    for args, match in [(dict(query=torch.zeros((1, 9, 5))), "channels"), (dict(heads=3), "heads"), (dict(views=[[0], [1]]), "views must be"),
                        (dict(views=[0]), "2 dimensions"), (dict(falloff=0.1), "do not lie"), (dict(cap=-1.0), "cap"),
                        (dict(num_query=[1, 1]), "one count per")]:
        call = dict(query=torch.zeros((1, 8, 5)), views=[[0, 1]]) | args
        with pytest.raises(ValueError, match=match):
            store.soft_match(call.pop("query"), call.pop("views"), **call)


def test_abi_refusals():
    """Bad sizes and missing workspaces come back as statuses before anything touches a device."""
    from pose_estimation_amd import _abi
    lib = _abi.lib

    def match(dtype=0, b=1, heads=1, d=64, dv=64, nq=10, cells=100, w=10, scale=1.0, cap=0.0, fall=None, ws=None, size=0, v=None):
        return lib.ispa_soft_match(1, 1, v, dtype, b, heads, d, dv, nq, cells, w, scale, cap, fall, None, None, None, 1, None, None, ws,
                                   size, None)

    for args, text in [(dict(dtype=2), b"dtype"), (dict(d=257), b"channels"), (dict(heads=0), b"channels"), (dict(cells=0), b"sizes"),
                       (dict(nq=-1), b"sizes"), (dict(cells=1 << 40), b"sizes"), (dict(b=1 << 20), b"sizes"), (dict(scale=math.nan), b"scale"),
                       (dict(cap=-1.0), b"cap"), (dict(fall=1, w=0), b"width"), (dict(dv=32), b"reference map is the value")]:
        assert match(**args) == -1 and text in lib.ispa_last_error(), args
    assert match(b=0) == 0 and match(nq=0) == 0
    need = lib.ispa_soft_match_workspace_bytes(0, 1, 1, 128, 128, 1, 1, 16384)
    assert need > 0 and lib.ispa_soft_match_workspace_bytes(0, 1, 1, 300, 128, 1, 1, 16384) == 0
    assert match(d=128, dv=128, nq=1, cells=16384) == -3 and b"workspace" in lib.ispa_last_error()
    assert match(d=128, dv=128, nq=1, cells=16384, ws=1, size=need - 1) == -3
    assert match(d=128, dv=128, nq=1, cells=16384, ws=1, size=need) == -1 and b"border" in lib.ispa_last_error()
    back = lambda **k: lib.ispa_soft_match_backward(1, 1, k.get("v"), 0, 1, 1, 64, 64, 10, 100, 10, 1.0, 0.0, None, None, None, None, 1, 1, 1,
                                                    None, 1, 1, k.get("dv"), None, 0, None)
    assert back(v=1) == -1 and b"come together" in lib.ispa_last_error()
    assert back() == -3 and b"workspace" in lib.ispa_last_error()
    assert lib.ispa_store_write(1, 0, None, 1, 2, 2, 4, 8, 16, 1, 1, 1, None) == -1 and b"kind" in lib.ispa_last_error()
    assert lib.ispa_store_write(1, 0, None, 1, -1, 0, 4, 8, 16, 1, 1, 1, None) == -1
    assert lib.ispa_store_read(None, 1, 1, 1, 2, 0, 4, 8, 16, 0, 1, None, None) == -1 and b"null" in lib.ispa_last_error()
    assert lib.ispa_store_match(1, 0, 1, 1, 1, 0, None, 2, 4, 1, 1, 64, 3, 100, 10, 1.0, 0.0, None, None, None, 1, None, None, 0,
                                None) == -1
