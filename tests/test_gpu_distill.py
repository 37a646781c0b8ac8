"""Top-logits distillation on the GPU against its definition in 64 bits.

Tolerances are error bounds.  A log-probability is a difference of two float32
numbers of the logits' size Z (over the temperature) and a sum of V exponentials,
each with an argument rounded at the size Z: it is within
d = (8 Z + V / 1024 + 32) 2^-24.  Probabilities have the relative error d, the
teacher's the same with its own Z and K, and the loss and its gradient follow by
their formulas; a rounding to the output's type comes on top."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0 ** -24
EPS = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def teacher_for(z, K, noise, g, lse, tau):
    t = z + noise * torch.randn(z.shape, device=DEV, generator=g)
    v, i = torch.topk(t, K, dim=1)
    perm = torch.randperm(K, device=DEV, generator=g)  # in no order
    return v[:, perm].contiguous(), i[:, perm].int().contiguous(), torch.logsumexp(t / tau, 1) if lse else None


def definition(logits, values, indices, lse, tau):
    """loss, d loss / d logits (64 bits) and bounds of their errors."""
    x = logits.double() / tau
    T, V = x.shape
    K = values.shape[1]
    live = (indices >= 0) & (indices < V)
    at = torch.where(live, indices.long(), 0)
    t = torch.where(live, values.double() / tau, -math.inf)
    lp = torch.log_softmax(x, 1)
    some = live.any(1, keepdim=True)
    n = lse.double()[:, None] if lse is not None else torch.where(some, torch.logsumexp(t, 1, keepdim=True), 0.0)
    q = torch.exp(t - n)
    lpk = lp.gather(1, at)
    loss = torch.where(q > 0, q * (t - n - lpk), 0.0).sum(1)
    Q = torch.zeros_like(x).scatter_add(1, at, q)
    p = lp.exp()
    zmax = x[x.isfinite()].abs().max().item() if x.isfinite().any() else 0.0
    tmax = t[t.isfinite()].abs().max().item() if t.isfinite().any() else 0.0
    d = (8 * zmax + V / 1024 + 32) * U
    dq = (8 * tmax + K + 32) * U
    spread = torch.where(q > 0, q * ((t - n).abs() + 1), 0.0).sum(1)
    lpsum = torch.where(q > 0, q * torch.where(lpk.isfinite(), lpk.abs(), 0.0), 0.0).sum(1)
    eloss = d * q.sum(1) + dq * (spread + lpsum) + K * U * (spread + lpsum)
    c = q.sum(1, keepdim=True)
    if lse is None:
        g = p * some - Q
        eg = d * p + dq * Q
    else:
        r = 1 - q.sum(1)
        r = torch.where(r > 1e-6, r, 0.0)
        listed = torch.zeros_like(x).scatter_add(1, at, live.double()) > 0
        unlisted = ~listed
        pr = torch.where(unlisted, p, 0.0).sum(1)
        loss = loss + torch.where(r > 0, r * (torch.log(r) - torch.log(pr)), 0.0)
        c = c + r[:, None]
        er = (dq + K * U) * q.sum(1) + 2 * U   # r is a difference from 1
        back = torch.where(r > 0, er * ((torch.log(r) - torch.log(pr)).abs() + 2) + r * (2 * d), er * 16)
        eloss = eloss + back
        share = torch.where(pr > 0, r / pr, 0.0)[:, None]
        g = p * c - Q - torch.where(unlisted, p * share, 0.0)
        eg = d * p * (c + 2 * share * unlisted) + dq * Q + p * (er[:, None] / torch.where(pr > 0, pr, 1.0)[:, None]) * unlisted + p * er[:, None]
    return loss, g / tau, 2 * eloss + 1e-7, 2 * eg / tau


def within(got, ref, bound, what):
    d = (got.double() - ref).abs()
    tol = bound + EPS[got.dtype] * (ref.abs() + bound) + TINY[got.dtype]
    bad = ~(d <= tol)
    if bad.any():
        i = int(bad.reshape(-1).nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off; first at {i}: "
                             f"{got.reshape(-1)[i].item()} for {ref.reshape(-1)[i].item()}, "
                             f"tolerance {tol.reshape(-1)[i].item()}")


SIZES = [(1, 1, 1), (1, 2, 1), (2, 3, 3), (5, 7, 2), (3, 8, 8), (4, 9, 4), (3, 64, 20), (2, 255, 16), (3, 1000, 100),
         (7, 4096, 64), (2, 8191, 1), (5, 32000, 256), (3, 50257, 64), (2, 131072, 1500)]


@pytest.mark.parametrize("T,V,K", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lse", [False, True])
def test_loss_and_gradient(bcjr_mod, T, V, K, dtype, lse):
    for tau in (1.0, 2.5, 0.6):
        g = gen(T + V + K)
        z = torch.randn(T, V, device=DEV, generator=g) * 2
        v, i, n = teacher_for(z, K, 0.7, g, lse, tau)
        logits = z.to(dtype).requires_grad_()
        up = torch.randn(T, device=DEV, generator=g)
        loss = bcjr_mod.topk_distill_loss(logits, v, i, temperature=tau, teacher_lse=n)
        (d,) = torch.autograd.grad(loss, logits, up)
        rl, rg, el, eg = definition(logits.detach(), v, i, n, tau)
        assert loss.dtype == torch.float32 and d.dtype == dtype
        within(loss, rl, el, "loss")
        ud = up.double()[:, None]
        within(d, rg * ud, eg * ud.abs(), "gradient")
        with torch.no_grad():
            assert torch.equal(bcjr_mod.topk_distill_loss(logits, v, i.long(), temperature=tau, teacher_lse=n), loss)
        l2, d2 = bcjr_mod.topk_distill_loss_and_grad(logits, v, i, up, temperature=tau, teacher_lse=n)
        assert torch.equal(l2, loss)
        within(d2, rg * ud, eg * ud.abs(), "gradient of one call")
        assert torch.equal(torch.autograd.grad(bcjr_mod.topk_distill_loss(logits, v, i, temperature=tau, teacher_lse=n),
                                               logits, up)[0], d), "a second gradient"


def test_peaked_student_keeps_its_rest(bcjr_mod):
    """The student's mass outside the entries is 1e-9 and less, the teacher's 0.1:
    1 - sum p would have none of it left."""
    T, V, K = 6, 5000, 8
    g = gen(9)
    z = torch.randn(T, V, device=DEV, generator=g)
    v, i = torch.topk(z, K, dim=1)
    z = z.scatter(1, i.long(), v + 30)
    n = torch.logsumexp(v, 1) - math.log(0.9)
    logits = z.requires_grad_()
    loss = bcjr_mod.topk_distill_loss(logits, v, i, teacher_lse=n)
    (d,) = torch.autograd.grad(loss.sum(), logits)
    rl, rg, el, eg = definition(logits.detach(), v, i, n, 1.0)
    within(loss, rl, el, "loss")
    within(d, rg, eg, "gradient")
    assert (rl > 1).all()


@pytest.mark.parametrize("lse", [False, True])
def test_difference_quotient(bcjr_mod, lse):
    """The loss along v: its third derivative is below 2 / tau^3 for |v| <= 1."""
    T, V, K, tau, h = 8, 600, 12, 1.5, 2.0 ** -5
    g = gen(10)
    z = torch.randn(T, V, device=DEV, generator=g) * 2
    v, i, n = teacher_for(z, K, 0.7, g, lse, tau)
    dirn = torch.randn(T, V, device=DEV, generator=g)
    dirn[:, ::3] += z.softmax(1)[:, ::3] * 30
    dirn = dirn / dirn.norm(dim=1, keepdim=True)
    logits = z.clone().requires_grad_()
    (d,) = torch.autograd.grad(bcjr_mod.topk_distill_loss(logits, v, i, temperature=tau, teacher_lse=n).sum(), logits)
    f = lambda x: bcjr_mod.topk_distill_loss(x, v, i, temperature=tau, teacher_lse=n).double()
    quot = (f(z + h * dirn) - f(z - h * dirn)) / (2 * h)
    el = definition(z, v, i, n, tau)[2]
    assert ((quot - (d.double() * dirn).sum(1)).abs() <= h * h / 6 * 2 / tau ** 3 * 2 + 2 * el / (2 * h) + 1e-6).all()


@pytest.mark.parametrize("lse", [False, True])
def test_missing_and_repeated_entries(bcjr_mod, lse):
    T, V, K = 6, 777, 10
    g = gen(12)
    z = torch.randn(T, V, device=DEV, generator=g)
    v, i, n = teacher_for(z, K, 0.5, g, lse, 1.0)
    i[0, 3:] = -1            # three entries
    i[1, :] = -1             # none
    i[2, 5] = V              # outside
    i[3, 4] = 2 ** 31 - 1
    i[4, 7] = i[4, 2]        # one twice
    v[5, 1] = -math.inf      # an entry without mass
    v[0, 5] = math.nan       # of an absent entry: not read
    logits = z.clone().requires_grad_()
    up = torch.rand(T, device=DEV, generator=g) + 0.5
    loss = bcjr_mod.topk_distill_loss(logits, v, i, teacher_lse=n)
    (d,) = torch.autograd.grad(loss, logits, up)
    vr = torch.where((i >= 0) & (i < V), v, 0.0)
    rl, rg, el, eg = definition(z, vr, i, n, 1.0)
    within(loss, rl, el, "loss")
    within(d, rg * up.double()[:, None], eg * up.double()[:, None], "gradient")
    assert abs(loss[1].item()) < 1e-6
    if not lse:
        assert loss[1].item() == 0 and (d[1] == 0).all()
    l2, d2 = bcjr_mod.topk_distill_loss_and_grad(logits, v, i, up, teacher_lse=n)
    assert torch.equal(l2, loss)
    within(d2, rg * up.double()[:, None], eg * up.double()[:, None], "gradient of one call")


def test_masked_vocabulary_infinities_and_nan(bcjr_mod):
    V, K = 100, 5
    g = gen(13)
    z = torch.randn(8, V, device=DEV, generator=g)
    v, i, _ = teacher_for(z, K, 0.1, g, False, 1.0)
    out = torch.ones(V, dtype=torch.bool, device=DEV)
    z[0, 50:] = -math.inf                      # masked vocabulary, entries in front of it
    i[0] = torch.arange(K, device=DEV)
    z[1, 50:] = torch.finfo(torch.float32).min  # the type's lowest value
    i[1] = torch.arange(K, device=DEV)
    z[2, i[2, 0].item()] = -math.inf           # an entry that the student gives nothing
    z[3, 7] = math.nan
    z[4, 7] = math.inf
    z[5] = -math.inf
    z[6] = math.nan                            # out of the loss: gradient 0
    logits = z.clone().requires_grad_()
    loss = bcjr_mod.topk_distill_loss(logits, v, i)
    up = torch.ones(8, device=DEV)
    up[6] = 0
    (d,) = torch.autograd.grad(loss, logits, up)
    ok = [0, 1, 7]
    rl, rg, el, eg = definition(z[ok], v[ok], i[ok], None, 1.0)
    within(loss[ok], rl, torch.full_like(el, 1e-5), "loss")
    within(d[ok], rg, torch.full_like(rg, 1e-6), "gradient")
    assert (d[0, 50:] == 0).all() and (d[1, 50:] == 0).all()
    assert loss[2].item() == math.inf and torch.isfinite(d[2]).all()
    assert loss[3:7].isnan().all()
    assert d[3].isnan().all() and d[5].isnan().all()
    assert (d[6] == 0).all()
    l2, d2 = bcjr_mod.topk_distill_loss_and_grad(logits, v, i, up)
    assert torch.equal(l2.nan_to_num(7.0, 8.0), loss.nan_to_num(7.0, 8.0)) and (d2[6] == 0).all()
    assert torch.isfinite(d2[ok]).all()
    # everything that has mass outside the entries is masked, the teacher has some there
    n = torch.logsumexp(v[:1], 1) + 0.1
    zz = torch.full((1, V), -math.inf, device=DEV)
    zz[0, :K] = 1.0
    zr = zz.requires_grad_()
    loss = bcjr_mod.topk_distill_loss(zr, v[:1], torch.arange(K, device=DEV)[None], teacher_lse=n)
    (d,) = torch.autograd.grad(loss.sum(), zr)
    assert loss.item() == math.inf and torch.isfinite(d).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides(bcjr_mod, dtype):
    """Row strides and starts that are not 16-byte aligned, and a transposed view."""
    T, K = 5, 6
    g = gen(14)
    for V, pad, first in [(1000, 24, 0), (1000, 24, 8), (1000, 3, 0), (1001, 3, 5), (333, 0, 0), (6, 5, 3), (1, 3, 1)]:
        wide = (torch.randn(T, V + pad, device=DEV, generator=g) * 2).to(dtype)
        first = min(first, pad)
        base = wide[:, first:first + V].contiguous()
        k = min(K, V)
        v, i, n = teacher_for(base.float(), k, 0.4, g, True, 1.0)
        up = torch.rand(T, device=DEV, generator=g)

        def both(x):
            x = x.detach().requires_grad_()
            loss = bcjr_mod.topk_distill_loss(x, v, i, teacher_lse=n)
            l2, d2 = bcjr_mod.topk_distill_loss_and_grad(x, v, i, up, teacher_lse=n)
            return loss.detach(), torch.autograd.grad(loss, x, up)[0], l2, d2

        rl, rg, el, eg = definition(base, v, i, n, 1.0)
        for x in (base, wide[:, first:first + V], base.t().contiguous().t()):
            l1, d1, l2, d2 = both(x)
            ud = up.double()[:, None]
            for l in (l1, l2):
                within(l, rl, el, (V, pad, first))
            for d in (d1, d2):
                within(d, rg * ud, eg * ud, (V, pad, first))
    # an expanded upstream gradient, as a mean gives
    x = base.detach().requires_grad_()
    (a,) = torch.autograd.grad(bcjr_mod.topk_distill_loss(x, v, i).mean(), x)
    (b,) = torch.autograd.grad(bcjr_mod.topk_distill_loss(x, v, i), x, torch.full((T,), 1 / T, device=DEV))
    assert torch.equal(a, b)


def test_empty_and_refusals(bcjr_mod):
    z = torch.zeros(4, 32, device=DEV)
    v, i = torch.zeros(4, 3, device=DEV), torch.zeros(4, 3, dtype=torch.int32, device=DEV)
    assert bcjr_mod.topk_distill_loss(z[:0], v[:0], i[:0]).shape == (0,)
    zr = z.clone().requires_grad_()
    loss = bcjr_mod.topk_distill_loss(zr, v[:, :0], i[:, :0])
    (d,) = torch.autograd.grad(loss.sum(), zr)
    assert (loss == 0).all() and (d == 0).all()
    with pytest.raises(AssertionError, match="temperature"):
        bcjr_mod.topk_distill_loss(z, v, i, temperature=0.0)
    with pytest.raises(AssertionError, match="\\(T, K\\)"):
        bcjr_mod.topk_distill_loss(z, v, i[:, :2])
    with pytest.raises(AssertionError, match="teacher_lse"):
        bcjr_mod.topk_distill_loss(z, v, i, teacher_lse=torch.zeros(3, device=DEV))
    with pytest.raises(AssertionError, match="row_weights"):
        bcjr_mod.topk_distill_loss_and_grad(z, v, i, torch.ones(3, device=DEV))
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        bcjr_mod.topk_distill_loss(z.double(), v, i)
    with pytest.raises(RuntimeError, match="int32 or int64"):
        bcjr_mod.topk_distill_loss(z, v, v)
    with pytest.raises(bcjr_mod._lib.BcjrError) as e:
        bcjr_mod.topk_distill_loss(z, v, i, temperature=math.inf)
    assert e.value.status == -1


def test_rows_past_32_bits(bcjr_mod):
    """Element offsets above 2^31 in logits and gradient: the last rows."""
    T, V, K = 16500, 131072, 4
    g = gen(15)
    logits = torch.zeros(T, V, device=DEV, dtype=torch.bfloat16)
    tail = torch.randn(3, V, device=DEV, generator=g)
    logits[-3:] = tail.bfloat16()
    v, i, n = teacher_for(tail, K, 0.5, g, True, 1.0)
    vv, ii, nn = v[:1].repeat(T, 1), i[:1].repeat(T, 1), n[:1].repeat(T)
    vv[-3:], ii[-3:], nn[-3:] = v, i, n
    w = torch.zeros(T, device=DEV)
    w[-3:] = 1
    rl, rg, el, eg = definition(logits[-3:], v, i, n, 1.0)
    x = logits.requires_grad_()
    loss = bcjr_mod.topk_distill_loss(x, vv, ii, teacher_lse=nn)
    (d,) = torch.autograd.grad(loss, x, w)
    within(loss[-3:], rl, el, "loss")
    within(d[-3:], rg, eg, "gradient")
    assert (d[:4] == 0).all()
    del d
    l2, d2 = bcjr_mod.topk_distill_loss_and_grad(x, vv, ii, w, teacher_lse=nn)
    within(d2[-3:], rg, eg, "gradient of one call")
    assert torch.equal(l2, loss)


def test_in_a_graph(bcjr_mod):
    T, V, K = 9, 3000, 16
    g = gen(16)
    z = torch.randn(T, V, device=DEV, generator=g)
    v, i, n = teacher_for(z, K, 0.5, g, True, 1.0)
    w = torch.rand(T, device=DEV, generator=g)
    buf = z.clone()
    bcjr_mod.topk_distill_loss_and_grad(buf, v, i, w, teacher_lse=n)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, d = bcjr_mod.topk_distill_loss_and_grad(buf, v, i, w, teacher_lse=n)
    for k in range(3):
        x = torch.randn(T, V, device=DEV, generator=g)
        want = bcjr_mod.topk_distill_loss_and_grad(x, v, i, w, teacher_lse=n)
        buf.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(loss, want[0]) and torch.equal(d, want[1]), k
