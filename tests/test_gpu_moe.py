"""Routing, grouped products and their sum on the GPU, against plain forms in
64 bits.

Tolerances are error bounds, element by element.  A float32 sum of n products in
any order is within (n + 2) 2^-24 sum |a b| of the sum; rounding to the output's
type adds 2^-8 (bfloat16) or 2^-11 (float16; 2^-25 below its normal range)
of the value.  Whole numbers, zeros and repeated calls are exact."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0 ** -24
EPS = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def within(got, ref, bound, what=""):
    """|got - ref| <= bound + one rounding to got's type, everywhere."""
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    d = (got.double() - ref).abs()
    tol = bound + EPS[got.dtype] * (ref.abs() + bound) + TINY[got.dtype]
    bad = ~(d <= tol)
    if bad.any():
        i = int(bad.reshape(-1).nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off; first at {i}: "
                             f"{got.reshape(-1)[i].item()} for {ref.reshape(-1)[i].item()}, "
                             f"tolerance {tol.reshape(-1)[i].item()}")


# -------------------------------------------------------------------- routing

def route_ref(logits, k, renormalize, valid):
    """By its definition, token by token, on the CPU in 64 bits."""
    l = logits.double().cpu()
    T, E = l.shape
    w = torch.zeros(T, k, dtype=torch.float64)
    ex = torch.full((T, k), -1, dtype=torch.int32)
    for t in range(T):
        if valid is not None and not bool(valid[t]):
            continue
        order = sorted(range(E), key=lambda e: (-l[t, e].item(), e))[:k]
        live = [e for e in order if l[t, e] > -math.inf]
        if not live:
            continue
        p = torch.softmax(l[t, live] if renormalize else l[t], 0)
        for j, e in enumerate(live):
            ex[t, j] = e
            w[t, j] = p[j] if renormalize else p[e]
    pairs = sorted((int(ex[t, j]), t, j) for t in range(T) for j in range(k) if ex[t, j] >= 0)
    rows = torch.full((T * k,), -1, dtype=torch.int32)
    slots = torch.full((T, k), -1, dtype=torch.int32)
    count = [0] * (E + 1)
    for n, (e, t, j) in enumerate(pairs):
        rows[n] = t
        slots[t, j] = n
        count[e + 1] += 1
    return w, ex, torch.tensor(count).cumsum(0).int(), rows, slots


ROUTES = [
    # T, E, k
    (1, 1, 1), (1, 64, 8), (3, 8, 8), (63, 7, 3), (64, 64, 8), (65, 64, 6), (256, 60, 4), (257, 64, 8),
    (300, 65, 2), (511, 128, 8), (700, 129, 16), (320, 256, 1), (290, 257, 8), (270, 1000, 9), (130, 64, 17),
    (260, 96, 64), (2049, 16, 2),
]


@pytest.mark.parametrize("T,E,k", ROUTES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("masked", [False, True])
def test_route(bcjr_mod, T, E, k, dtype, masked):
    g = gen(T * 1000 + E + k)
    # steps of 1/4 in a narrow range: many ties
    l = (torch.randn(T, E, device=DEV, generator=g) * 6).round().div(4).to(dtype)
    valid = None
    if masked:
        l[torch.rand(T, E, device=DEV, generator=g) < 0.3] = -math.inf
        l[torch.rand(T, device=DEV, generator=g) < 0.1] = -math.inf
        valid = torch.rand(T, device=DEV, generator=g) >= 0.2
    for norm in (False, True):
        lg = l.detach().clone().requires_grad_()
        r = bcjr_mod.moe_route(lg, k, renormalize=norm, valid=valid)
        w, ex, off, rows, slots = route_ref(l, k, norm, valid)
        for name, a, b in (("experts", r.experts, ex), ("offsets", r.offsets, off), ("rows", r.rows, rows),
                           ("slots", r.slots, slots)):
            assert a.dtype == torch.int32 and torch.equal(a.cpu(), b), (name, norm)
        # exp of arguments within 16 (log2 units within 23): 2 ulp of the argument, and E terms
        rel = (2 * 24 + E + 8) * U
        within(r.weights, w.to(DEV), rel * w.to(DEV), "weights")
        up = torch.randn(T, k, device=DEV, generator=g)
        (gl,) = torch.autograd.grad(r.weights, lg, up)
        assert gl.dtype == dtype
        with torch.enable_grad():
            ld = l.double().cpu().requires_grad_()
            live = ex >= 0
            at = ex.clamp(min=0).long()
            if norm:
                z = torch.where(live, ld.gather(1, at), -math.inf)
                p = torch.softmax(torch.where(live.any(1, keepdim=True), z, 0.0), 1)
            else:
                some = (ld.detach() > -math.inf).any(1, keepdim=True)
                p = torch.softmax(torch.where(some, ld, 0.0), 1).gather(1, at)
            (ref,) = torch.autograd.grad((torch.where(live, p, 0.0) * up.double().cpu()).sum(), ld)
        # both terms of the difference, each with the weights' error
        mag = (w * up.double().cpu().abs()).sum(1, keepdim=True).to(DEV)
        within(gl, ref.to(DEV), 4 * rel * (mag + ref.to(DEV).abs()), "logits' gradient")


def test_route_difference_quotient(bcjr_mod):
    """<gradient, v> against (f(l + hv) - f(l - hv)) / 2h, f = sum u w: the third
    derivative of a softmax component is below 1, so with |v| <= 1 the quotient
    is within |u|_1 h^2 / 6 + 2 |u|_1 delta / 2h."""
    g = gen(5)
    T, E, k, h = 40, 24, 4, 2.0 ** -6
    l = torch.randn(T, E, device=DEV, generator=g) * 3
    v = torch.randn(T, E, device=DEV, generator=g)
    v = v / v.norm(dim=1, keepdim=True)
    up = torch.randn(T, k, device=DEV, generator=g)
    for norm in (False, True):
        x = l.clone().requires_grad_()
        r = bcjr_mod.moe_route(x, k, renormalize=norm)
        (gl,) = torch.autograd.grad(r.weights, x, up)
        lo, hi = bcjr_mod.moe_route(l - h * v, k, renormalize=norm), bcjr_mod.moe_route(l + h * v, k, renormalize=norm)
        same = (lo.experts == r.experts).all(1) & (hi.experts == r.experts).all(1)
        assert same.float().mean() > 0.5
        quot = ((hi.weights - lo.weights).double() * up).sum(1) / (2 * h)
        d = (quot - (gl.double() * v).sum(1)).abs()
        u1 = up.abs().double().sum(1)
        assert (d[same] <= (u1 * (h * h / 6 * 6 + (2 * 24 + E + 8) * U / h))[same]).all()


def test_route_nan_and_infinities(bcjr_mod):
    inf, nan = math.inf, math.nan
    l = torch.tensor([[0.0, nan, 2.0, -inf], [inf, 1.0, inf, 0.0], [-inf] * 4, [-0.0, 0.0, -0.0, 0.0],
                      [nan] * 4, [-nan, 3.0, 1.0, 2.0]], device=DEV)
    low = torch.finfo(torch.float32).min
    l = torch.cat([l, torch.tensor([[low, low, -inf, low]], device=DEV)])
    r = bcjr_mod.moe_route(l, 3)
    assert r.experts.tolist() == [[1, 2, 0], [0, 2, 1], [-1, -1, -1], [0, 1, 2], [0, 1, 2], [0, 1, 3], [0, 1, 3]]
    w = r.weights.cpu()
    assert w[0].isnan().all() and w[4].isnan().all() and w[5].isnan().all()
    assert w[1].isnan().any()
    assert (w[2] == 0).all() and torch.allclose(w[3], torch.full((3,), 0.25))
    assert torch.allclose(w[6], torch.full((3,), 1 / 3))
    assert (r.slots[2] == -1).all() and int(r.offsets[-1]) == 18


def test_route_strides_empty_and_lead(bcjr_mod):
    g = gen(11)
    wide = torch.randn(50, 100, device=DEV, generator=g)
    a, b = bcjr_mod.moe_route(wide[:, 3:40], 5), bcjr_mod.moe_route(wide[:, 3:40].contiguous(), 5)
    c = bcjr_mod.moe_route(wide[:, 3:40].t().contiguous().t(), 5)
    for x, y, z in zip(a, b, c):
        assert torch.equal(x, y) and torch.equal(x, z)
    none = bcjr_mod.moe_route(torch.empty(0, 8, device=DEV), 2)
    assert none.offsets.tolist() == [0] * 9 and none.rows.numel() == 0 and none.weights.shape == (0, 2)


def test_route_large_is_sorted(bcjr_mod):
    """Many tokens, several words a block: the order by its properties."""
    g = gen(12)
    T, E, k = 40000, 48, 6
    l = torch.randn(T, E, device=DEV, generator=g)
    r = bcjr_mod.moe_route(l, k)
    M = T * k
    assert int(r.offsets[0]) == 0 and int(r.offsets[-1]) == M
    flat = r.experts.reshape(-1).long()
    assert torch.equal(torch.bincount(flat, minlength=E), (r.offsets[1:] - r.offsets[:-1]).long())
    order = torch.sort(flat, stable=True)[1]
    assert torch.equal(r.rows.long(), order // k)
    assert torch.equal(r.slots.reshape(-1)[order].long(), torch.arange(M, device=DEV))
    assert torch.equal(r.experts, bcjr_mod.moe_route(l, k).experts)


# ----------------------------------------------------------- grouped products

def groups_of(M, E, style, g):
    """offsets (E + 1,) int32: `style` says how M rows are shared."""
    if style == "one":          # all rows with one expert
        c = torch.zeros(E, dtype=torch.long)
        c[E // 2] = M
    elif style == "even":
        c = torch.full((E,), M // E)
        c[: M % E] += 1
    elif style == "short":      # a tenth of the rows has no expert
        c = torch.bincount(torch.randint(0, E, (M - M // 10,), generator=g), minlength=E)
    else:                       # skewed, empty experts among them
        p = torch.rand(E, generator=g) ** 4
        p[torch.rand(E, generator=g) < 0.2] = 0
        p[0] += 1e-3
        c = torch.bincount(torch.multinomial(p, M, True, generator=g), minlength=E) if M else torch.zeros(E)
    o = torch.zeros(E + 1, dtype=torch.int32)
    o[1:] = c.cumsum(0)
    return o.to(DEV)


def product_ref(x, w, offsets, rows=None, gy=None):
    """y, dx by place, dw and the sums of magnitudes of their products."""
    o = offsets.tolist()
    E, N, K = w.shape
    xr = x.double() if rows is None else torch.cat([x, x.new_zeros(1, K)])[rows.long()].double()
    M = xr.shape[0]
    y, my = (torch.zeros(M, N, device=DEV, dtype=torch.float64) for _ in range(2))
    out = [y, my]
    if gy is not None:
        dx, mx = (torch.zeros(M, K, device=DEV, dtype=torch.float64) for _ in range(2))
        dw, mw = (torch.zeros(E, N, K, device=DEV, dtype=torch.float64) for _ in range(2))
        out += [dx, mx, dw, mw]
    wd = w.double()
    for e in range(E):
        s = slice(o[e], o[e + 1])
        y[s], my[s] = xr[s] @ wd[e].t(), xr[s].abs() @ wd[e].t().abs()
        if gy is not None:
            gd = gy[s].double()
            dx[s], mx[s] = gd @ wd[e], gd.abs() @ wd[e].abs()
            dw[e], mw[e] = gd.t() @ xr[s], gd.t().abs() @ xr[s].abs()
    return out


PRODUCTS = [
    # M, E, N, K, style
    (1, 1, 1, 1, "one"), (1, 8, 64, 64, "one"), (5, 3, 7, 9, "skew"), (16, 4, 16, 32, "even"), (33, 64, 48, 40, "skew"),
    (100, 5, 333, 517, "skew"), (128, 2, 128, 128, "even"), (257, 3, 264, 136, "skew"), (300, 7, 256, 512, "short"),
    (513, 4, 130, 66, "even"), (700, 3, 520, 72, "one"), (1000, 130, 72, 80, "skew"), (1200, 2, 256, 256, "even"),
    (2000, 16, 384, 192, "skew"), (640, 8, 2048, 1024, "skew"), (3000, 6, 1000, 88, "short"), (90, 64, 512, 2048, "skew"),
]


@pytest.mark.parametrize("M,E,N,K,style", PRODUCTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_grouped_forward_backward(bcjr_mod, M, E, N, K, style, dtype):
    g = torch.Generator()
    g.manual_seed(M + N)
    gd = gen(M * 7 + K)
    off = groups_of(M, E, style, g)
    x = torch.randn(M, K, device=DEV, generator=gd).to(dtype).requires_grad_()
    gy = torch.randn(M, N, device=DEV, generator=gd).to(dtype)
    for wtype in (dtype, torch.float32):
        w = (torch.randn(E, N, K, device=DEV, generator=gd) / 8).to(wtype).requires_grad_()
        y = bcjr_mod.grouped_matmul(x, w, off)
        gx, gw = torch.autograd.grad(y, (x, w), gy)
        assert y.dtype == gx.dtype == dtype and gw.dtype == wtype
        ry, my, rx, mx, rw, mw = product_ref(x.detach(), w.detach().to(dtype), off, gy=gy)
        within(y, ry, (K + 2) * U * my, "y")
        within(gx, rx, (N + 2) * U * mx, "gx")
        within(gw, rw, (M + 2) * U * mw, "gw")
        with torch.no_grad():
            assert torch.equal(bcjr_mod.grouped_matmul(x, w, off), y), "a second call"
        assert torch.equal(torch.autograd.grad(bcjr_mod.grouped_matmul(x, w, off), w, gy)[0], gw), "a second gradient"


@pytest.mark.parametrize("T,E,k,N,K", [(1, 8, 2, 64, 64), (4, 64, 8, 256, 512), (37, 9, 3, 56, 120), (150, 7, 2, 333, 517),
                                       (600, 16, 4, 256, 128), (900, 5, 2, 264, 320)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gathered_rows(bcjr_mod, T, E, k, N, K, dtype):
    """Rows through a routing in which some tokens have fewer experts or none."""
    g = gen(T + N)
    l = torch.randn(T, E, device=DEV, generator=g)
    l[torch.rand(T, E, device=DEV, generator=g) < 0.5] = -math.inf
    r = bcjr_mod.moe_route(l, k)
    M = T * k
    x = torch.randn(T, K, device=DEV, generator=g).to(dtype).requires_grad_()
    w = (torch.randn(E, N, K, device=DEV, generator=g) / 8).requires_grad_()
    gy = torch.randn(M, N, device=DEV, generator=g).to(dtype)
    y = bcjr_mod.grouped_matmul(x, w, r.offsets, rows=r.rows, slots=r.slots)
    gx, gw = torch.autograd.grad(y, (x, w), gy)
    ry, my, rx, mx, rw, mw = product_ref(x.detach(), w.detach().to(dtype), r.offsets, r.rows, gy)
    within(y, ry, (K + 2) * U * my, "y")
    within(gw, rw, (M + 2) * U * mw, "gw")
    # a place's gradient is rounded to the rows' type, then a row's places are summed
    place = (N + 2) * U * mx
    place = place + EPS[dtype] * (rx.abs() + place) + TINY[dtype]
    s = r.slots.long()
    live = (s >= 0)[..., None]
    pick = lambda a: torch.where(live, a[s.clamp(min=0)], 0.0).sum(1)
    within(gx, pick(rx), pick(place) + (k + 2) * U * pick(rx.abs() + place), "gx")
    live_rows = int(r.offsets[-1])
    assert (y[live_rows:] == 0).all()


@pytest.mark.parametrize("N,K,style", [(1032, 1160, "skew"), (1160, 1032, "even"), (1033, 1161, "short")])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_grouped_many_rows(bcjr_mod, N, K, style, dtype):
    """Rows and tiles enough for the largest tiles, forward and backward."""
    test_grouped_forward_backward(bcjr_mod, 20000, 40, N, K, style, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gathered_many_rows(bcjr_mod, dtype):
    test_gathered_rows(bcjr_mod, 5000, 40, 4, 1032, 1160, dtype)


@pytest.mark.parametrize("M,N,K", [(60, 700, 1600), (200, 1600, 700), (1500, 1600, 700), (4000, 1600, 1700)])
def test_grouped_same_bits_beside_other_sizes(bcjr_mod, M, N, K):
    """A row's product does not depend on how many rows its call has, nor on the tiles that it is cut into."""
    g = gen(M)
    E = 20
    x = torch.randn(M, K, device=DEV, generator=g).bfloat16()
    w = torch.randn(E, N, K, device=DEV, generator=g).bfloat16()
    gc = torch.Generator()
    gc.manual_seed(M)
    off = groups_of(M, E, "even", gc)
    y = bcjr_mod.grouped_matmul(x, w, off)
    e = E // 2
    a, b = int(off[e]), int(off[e + 1])
    alone = bcjr_mod.grouped_matmul(x[a:b], w[e:e + 1], torch.tensor([0, b - a], dtype=torch.int32, device=DEV))
    assert torch.equal(alone, y[a:b])


def test_places_without_expert_do_not_leak(bcjr_mod):
    """NaN in rows behind the last group reach neither y nor the gradients."""
    M, E, N, K = 200, 4, 96, 160
    off = torch.tensor([0, 40, 40, 90, 130], dtype=torch.int32, device=DEV)
    g = gen(3)
    x = torch.randn(M, K, device=DEV, generator=g).bfloat16()
    gy = torch.randn(M, N, device=DEV, generator=g).bfloat16()
    x[130:] = math.nan
    gy[130:] = math.inf
    x.requires_grad_()
    w = torch.randn(E, N, K, device=DEV, generator=g).requires_grad_()
    y = bcjr_mod.grouped_matmul(x, w, off)
    gx, gw = torch.autograd.grad(y, (x, w), gy)
    assert (y[130:] == 0).all() and (gx[130:] == 0).all()
    assert torch.isfinite(y).all() and torch.isfinite(gx).all() and torch.isfinite(gw).all()
    assert (gw[1] == 0).all() and (gw[0] != 0).any()


def test_neighbours_do_not_leak(bcjr_mod):
    """NaN in one expert's rows and weights stay with it, where tiles are ragged."""
    for K in (160, 161):
        M, E, N = 150, 3, 200
        off = torch.tensor([0, 37, 81, 150], dtype=torch.int32, device=DEV)
        g = gen(4)
        x = torch.randn(M, K, device=DEV, generator=g).half()
        w = torch.randn(E, N, K, device=DEV, generator=g).half()
        gy = torch.randn(M, N, device=DEV, generator=g).half()
        x[37:81] = math.nan
        w[1] = math.nan
        gy[37:81] = math.nan
        x.requires_grad_(), w.requires_grad_()
        y = bcjr_mod.grouped_matmul(x, w, off)
        gx, gw = torch.autograd.grad(y, (x, w), gy)
        for t in (y, gx):
            assert torch.isfinite(t[:37]).all() and torch.isfinite(t[81:]).all() and t[37:81].isnan().all()
        assert torch.isfinite(gw[[0, 2]]).all() and gw[1].isnan().all()


@pytest.mark.parametrize("M,E,N,K", [(3, 4, 24, 16), (100, 4, 64, 96), (100, 4, 33, 35), (600, 3, 256, 128)])
def test_grouped_difference(bcjr_mod, M, E, N, K):
    """Whole numbers, so that every sum is exact: L = <gy, y> grows by exactly
    <gx, v> and <gw, v> when x and w grow by v (the product is linear in each)."""
    g = gen(M)
    ints = lambda *s: torch.randint(-1, 2, s, device=DEV, generator=g).to(torch.float16)
    gc = torch.Generator()
    gc.manual_seed(M)
    off = groups_of(M, E, "short", gc)
    x, w, gy = ints(M, K), ints(E, N, K), ints(M, N)
    vx, vw = ints(M, K), ints(E, N, K)
    f = lambda a, b: (gy.double() * bcjr_mod.grouped_matmul(a, b, off).double()).sum().item()
    xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
    gx, gw = torch.autograd.grad(bcjr_mod.grouped_matmul(xr, wr, off), (xr, wr), gy)
    assert f(x + vx, w) - f(x, w) == (gx.double() * vx.double()).sum().item()
    assert f(x, w + vw) - f(x, w) == (gw.double() * vw.double()).sum().item()


def test_grouped_strides_and_types(bcjr_mod):
    g = gen(21)
    M, E, N, K = 100, 3, 64, 128
    off = torch.tensor([0, 30, 64, 100], device=DEV)  # int64
    wide = torch.randn(M, 3 * K, device=DEV, generator=g).bfloat16()
    w = torch.randn(E, N, K, device=DEV, generator=g).bfloat16()
    base = bcjr_mod.grouped_matmul(wide[:, K:2 * K].contiguous(), w, off.int())
    for x in (wide[:, K:2 * K], wide[:, K:2 * K].t().contiguous().t()):
        assert torch.equal(bcjr_mod.grouped_matmul(x, w, off), base)
    odd = torch.empty(M, 2 * K + 3, device=DEV).bfloat16()  # rows that are not 16-byte aligned
    odd[:, 1:K + 1] = wide[:, K:2 * K]
    y = bcjr_mod.grouped_matmul(odd[:, 1:K + 1], w, off)
    ry, my = product_ref(wide[:, K:2 * K], w, off)
    within(y, ry, (K + 2) * U * my)
    wt = w.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(bcjr_mod.grouped_matmul(wide[:, K:2 * K], wt, off), base)
    # a gradient that is one row, expanded
    x = wide[:, K:2 * K].contiguous().requires_grad_()
    wr = w.clone().requires_grad_()
    one = torch.randn(1, N, device=DEV, generator=g).bfloat16()
    a = torch.autograd.grad(bcjr_mod.grouped_matmul(x, wr, off), (x, wr), one.expand(M, N))
    b = torch.autograd.grad(bcjr_mod.grouped_matmul(x, wr, off), (x, wr), one.expand(M, N).contiguous())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_grouped_empty(bcjr_mod):
    w = torch.randn(3, 8, 16, device=DEV).bfloat16().requires_grad_()
    x = torch.empty(0, 16, device=DEV).bfloat16().requires_grad_()
    y = bcjr_mod.grouped_matmul(x, w, torch.zeros(4, dtype=torch.int32, device=DEV))
    assert y.shape == (0, 8)
    gx, gw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert gx.shape == (0, 16) and (gw == 0).all()
    # rows, and no expert has any
    x = torch.randn(20, 16, device=DEV).bfloat16()
    assert (bcjr_mod.grouped_matmul(x, w.detach(), torch.zeros(4, dtype=torch.int32, device=DEV)) == 0).all()


def test_grouped_offsets_out_of_range(bcjr_mod):
    """Offsets above M are clamped to it, places outside [0, T) are rows of zeros."""
    g = gen(8)
    x = torch.randn(50, 64, device=DEV, generator=g).bfloat16()
    w = torch.randn(2, 32, 64, device=DEV, generator=g).bfloat16()
    off = torch.tensor([0, 20, 10 ** 6], dtype=torch.int32, device=DEV)
    ok = torch.tensor([0, 20, 50], dtype=torch.int32, device=DEV)
    assert torch.equal(bcjr_mod.grouped_matmul(x, w, off), bcjr_mod.grouped_matmul(x, w, ok))
    rows = torch.arange(50, dtype=torch.int32, device=DEV)
    rows[5], rows[30] = -7, 10 ** 6
    y = bcjr_mod.grouped_matmul(x, w, ok, rows=rows)
    x0 = x.clone()
    x0[[5, 30]] = 0
    assert torch.equal(y, bcjr_mod.grouped_matmul(x0, w, ok))


def test_grouped_refusals(bcjr_mod):
    x, w = torch.zeros(4, 16, device=DEV).bfloat16(), torch.zeros(2, 8, 16, device=DEV).bfloat16()
    off = torch.zeros(3, dtype=torch.int32, device=DEV)
    with pytest.raises(AssertionError, match="E\\+1=3"):
        bcjr_mod.grouped_matmul(x, w, off[:2])
    with pytest.raises(AssertionError, match="x must be"):
        bcjr_mod.grouped_matmul(x[:, :8], w, off)
    with pytest.raises(AssertionError, match="or float32"):
        bcjr_mod.grouped_matmul(x, w.half(), off)
    with pytest.raises(bcjr_mod._lib.BcjrError, match="bfloat16 and float16") as e:
        bcjr_mod.grouped_matmul(x.float(), w.float(), off)
    assert e.value.status == -2
    rows = torch.zeros(4, dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError, match="needs slots"):
        bcjr_mod.grouped_matmul(x.requires_grad_(), w, off, rows=rows)


def test_grouped_long_rows(bcjr_mod):
    """Element offsets above 2^31: the last group's rows."""
    M, K, N = 33000, 65600, 16
    x = torch.zeros(M, K, device=DEV, dtype=torch.bfloat16)
    g = gen(2)
    x[-70:] = torch.randn(70, K, device=DEV, generator=g).bfloat16()
    w = torch.randn(2, N, K, device=DEV, generator=g).bfloat16()
    off = torch.tensor([0, M - 60, M], dtype=torch.int32, device=DEV)
    gy = torch.zeros(M, N, device=DEV, dtype=torch.bfloat16)
    gy[-70:] = torch.randn(70, N, device=DEV, generator=g).bfloat16()
    xr, wr = x.requires_grad_(), w.requires_grad_()
    y = bcjr_mod.grouped_matmul(xr, wr, off)
    gx, gw = torch.autograd.grad(y, (xr, wr), gy)
    sub = torch.tensor([0, 10, 70], dtype=torch.int32, device=DEV)
    ry, my, rx, mx, rw, mw = product_ref(x.detach()[-70:], w.detach(), sub, gy=gy[-70:])
    within(y[-70:], ry, (K + 2) * U * my)
    within(gx[-70:], rx, (N + 2) * U * mx)
    within(gw, rw, (72) * U * mw)
    assert (y[:-70] == 0).all()


# -------------------------------------------------------------------- combine

@pytest.mark.parametrize("T,E,k,N", [(1, 4, 1, 1), (1, 8, 8, 2048), (7, 5, 3, 33), (40, 16, 4, 200), (65, 8, 2, 4100),
                                     (9, 70, 66, 24)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_combine(bcjr_mod, T, E, k, N, dtype):
    g = gen(T + N)
    M = T * k
    # a routing by hand (k may pass the router's 64): some pairs have no place
    slots = torch.randperm(M, device=DEV, generator=g).reshape(T, k).int()
    dead = torch.rand(T, k, device=DEV, generator=g) < 0.2
    gone = int(dead.sum())
    rows = torch.full((M,), -1, dtype=torch.int32, device=DEV)
    slots = torch.where(dead, -1, torch.argsort(torch.argsort(torch.where(dead, M + 1, slots).reshape(-1))).reshape(T, k)).int()
    live = slots >= 0
    rows[slots[live].long()] = torch.arange(T, device=DEV, dtype=torch.int32)[:, None].expand(T, k)[live]
    y = torch.randn(M, N, device=DEV, generator=g).to(dtype)
    y[M - gone:] = math.nan
    y.requires_grad_()
    w = torch.rand(T, k, device=DEV, generator=g).requires_grad_()
    go = torch.randn(T, N, device=DEV, generator=g).to(dtype)
    out = bcjr_mod.moe_combine(y, w, rows, slots)
    gy, gw = torch.autograd.grad(out, (y, w), go)
    s = slots.clamp(min=0).long()
    yd = torch.where(live[..., None], y.detach().double()[s], 0.0)
    wd, gd = w.detach().double(), go.double()
    within(out, (wd[..., None] * yd).sum(1), (k + 2) * U * (wd[..., None] * yd).abs().sum(1), "out")
    ref = torch.zeros(M, N, dtype=torch.float64, device=DEV)
    ref[slots[live].long()] = (wd[..., None] * gd[:, None])[live]
    within(gy, ref, 2 * U * ref.abs(), "gy")
    within(gw, (yd * gd[:, None]).sum(2), (N + 2) * U * (yd * gd[:, None]).abs().sum(2), "gweights")
    assert (gy[M - gone:] == 0).all()


def test_combine_strides_refusals_and_empty(bcjr_mod):
    g = gen(31)
    T, k, N = 12, 2, 64
    wide = torch.randn(T * k, 3 * N + 1, device=DEV, generator=g).bfloat16()
    slots = torch.arange(T * k, device=DEV, dtype=torch.int32).reshape(T, k)
    rows = torch.arange(T, device=DEV, dtype=torch.int32).repeat_interleave(k)
    w = torch.rand(T, k, device=DEV, generator=g)
    base = bcjr_mod.moe_combine(wide[:, N:2 * N].contiguous(), w, rows, slots)
    assert torch.equal(bcjr_mod.moe_combine(wide[:, N:2 * N], w, rows, slots), base)
    assert torch.equal(bcjr_mod.moe_combine(wide[:, N:2 * N], w.t().contiguous().t(), rows, slots.long()), base)
    # the gradient of a broadcast: an expanded row
    y = wide[:, N:2 * N].contiguous().requires_grad_()
    wr = w.clone().requires_grad_()
    one = torch.randn(1, N, device=DEV, generator=g).bfloat16()
    a = torch.autograd.grad(bcjr_mod.moe_combine(y, wr, rows, slots), (y, wr), one.expand(T, N))
    b = torch.autograd.grad(bcjr_mod.moe_combine(y, wr, rows, slots), (y, wr), one.expand(T, N).contiguous())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    with pytest.raises(AssertionError, match="all must be"):
        bcjr_mod.moe_combine(y[:-1], w, rows, slots)
    with pytest.raises(AssertionError, match="weights and slots"):
        bcjr_mod.moe_combine(y, w[:, :1], rows, slots)
    empty = bcjr_mod.moe_combine(y[:0].detach(), w[:0], rows[:0], slots[:0])
    assert empty.shape == (0, N)


def test_combine_difference(bcjr_mod):
    """Linear in y and in the weights; whole numbers, so the differences are exact."""
    g = gen(32)
    T, k, N = 30, 3, 40
    ints = lambda *s: torch.randint(-2, 3, s, device=DEV, generator=g).float()
    slots = torch.randperm(T * k, device=DEV, generator=g).reshape(T, k).int()
    rows = torch.empty(T * k, dtype=torch.int32, device=DEV)
    rows[slots.long()] = torch.arange(T, device=DEV, dtype=torch.int32)[:, None].expand(T, k)
    y, w, go, vy, vw = ints(T * k, N), ints(T, k), ints(T, N), ints(T * k, N), ints(T, k)
    yr, wr = y.clone().requires_grad_(), w.clone().requires_grad_()
    gy, gw = torch.autograd.grad(bcjr_mod.moe_combine(yr, wr, rows, slots), (yr, wr), go)
    f = lambda a, b: (go * bcjr_mod.moe_combine(a, b, rows, slots)).sum().item()
    assert f(y + vy, w) - f(y, w) == (gy * vy).sum().item()
    assert f(y, w + vw) - f(y, w) == (gw * vw).sum().item()


# ------------------------------------------------------------------- together

def _layer(b, x, router, wgu, wd, k):
    r = b.moe_route(x.float() @ router.t(), k, renormalize=True)
    h = b.grouped_matmul(x, wgu, r.offsets, rows=r.rows, slots=r.slots)
    gate, up = h.chunk(2, 1)
    y = b.grouped_matmul(torch.nn.functional.silu(gate) * up, wd, r.offsets)
    return b.moe_combine(y, r.weights, r.rows, r.slots)


def test_layer_on_another_stream_and_in_a_graph(bcjr_mod):
    g = gen(41)
    T, E, k, H, I = 48, 8, 2, 128, 96
    x = torch.randn(T, H, device=DEV, generator=g).bfloat16()
    router = torch.randn(E, H, device=DEV, generator=g) / 8
    wgu = (torch.randn(E, 2 * I, H, device=DEV, generator=g) / 8).bfloat16()
    wd = (torch.randn(E, H, I, device=DEV, generator=g) / 8).bfloat16()
    want = _layer(bcjr_mod, x, router, wgu, wd, k)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = _layer(bcjr_mod, x, router, wgu, wd, k)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    buf = x.clone()
    with torch.cuda.graph(graph):
        out = _layer(bcjr_mod, buf, router, wgu, wd, k)
    for i in range(4):
        xi = torch.randn(T, H, device=DEV, generator=g).bfloat16()
        want = _layer(bcjr_mod, xi, router, wgu, wd, k)
        buf.copy_(xi)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i


def test_layer_trains_quantized_experts(bcjr_mod):
    """Gradients reach the latent weights of bcjr_quantize_experts and the router."""
    g = gen(42)
    T, E, k, H, I = 24, 4, 2, 64, 32
    cb = bcjr_mod.make_1mad_codebook(10, DEV)
    lat = [(torch.randn(*s, device=DEV, generator=g) / 8).requires_grad_() for s in [(2 * I, H)] * E + [(H, I)] * E]
    sl = [torch.ones(w.shape[0], device=DEV) for w in lat]
    sr = [torch.ones(w.shape[1], device=DEV) for w in lat]
    q = bcjr_mod.bcjr_quantize_experts(lat, sl, sr, cb, 0.3, L=10, k=2, V=1)
    router = (torch.randn(E, H, device=DEV, generator=g) / 8).requires_grad_()
    x = torch.randn(T, H, device=DEV, generator=g).bfloat16()
    out = _layer(bcjr_mod, x, router, torch.stack(q[:E]), torch.stack(q[E:]), k)
    out.float().square().sum().backward()
    for t in lat + [router]:
        assert t.grad is not None and torch.isfinite(t.grad).all() and (t.grad != 0).any()


def test_layer_compiles_whole(bcjr_mod):
    """torch.compile traces a layer's forward and backward without a graph break."""
    g = gen(43)
    T, E, k, H, I = 40, 6, 2, 64, 48
    x = torch.randn(T, H, device=DEV, generator=g).bfloat16().requires_grad_()
    router = torch.randn(E, H, device=DEV, generator=g) / 8
    wgu = (torch.randn(E, 2 * I, H, device=DEV, generator=g) / 8).requires_grad_()
    wd = (torch.randn(E, H, I, device=DEV, generator=g) / 8).requires_grad_()
    idx = torch.randint(0, H, (T, 5), device=DEV, generator=g)
    val = torch.randn(T, 5, device=DEV, generator=g)

    def step(x, wgu, wd):
        out = _layer(bcjr_mod, x, router, wgu, wd, k)
        return bcjr_mod.topk_distill_loss(out, val, idx, temperature=2.0).mean()

    want = step(x, wgu, wd)
    gw = torch.autograd.grad(want, (x, wgu, wd))
    got = torch.compile(step, fullgraph=True, backend="aot_eager")(x, wgu, wd)
    gg = torch.autograd.grad(got, (x, wgu, wd))
    assert torch.equal(got, want)
    for a, b in zip(gg, gw):
        assert torch.equal(a, b)


def test_gradients_of_one_input(bcjr_mod):
    """Gradients of the rows alone, of the weights alone, and none."""
    g = gen(44)
    off = torch.tensor([0, 5, 12], dtype=torch.int32, device=DEV)
    x = torch.randn(12, 40, device=DEV, generator=g).half()
    w = torch.randn(2, 24, 40, device=DEV, generator=g)
    gy = torch.randn(12, 24, device=DEV, generator=g).half()
    xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
    gx, gw = torch.autograd.grad(bcjr_mod.grouped_matmul(xr, wr, off), (xr, wr), gy)
    assert torch.equal(torch.autograd.grad(bcjr_mod.grouped_matmul(xr, w, off), xr, gy)[0], gx)
    assert torch.equal(torch.autograd.grad(bcjr_mod.grouped_matmul(x, wr, off), wr, gy)[0], gw)
    assert not bcjr_mod.grouped_matmul(x, w, off).requires_grad


@pytest.mark.parametrize("n,ld,dtype,to", [(1, 1, torch.float32, torch.bfloat16), (7, 9, torch.float32, torch.float16),
                                           (8, 8, torch.float16, torch.float16), (517, 517, torch.bfloat16, torch.bfloat16),
                                           (333, 340, torch.float16, torch.float16), (1024, 1024, torch.float32, torch.bfloat16)])
def test_padded_copy(bcjr_mod, n, ld, dtype, to):
    x = torch.randn(37, ld, device=DEV, generator=gen(n)).to(dtype)[:, :n]
    out = bcjr_mod.moe._ops.pad_rows(x, torch.empty(0, device=DEV, dtype=to))
    assert out.shape == x.shape and out.stride(0) == (n + 7) // 8 * 8 and torch.equal(out, x.to(to))
    whole = torch.as_strided(out, (37, out.stride(0)), (out.stride(0), 1))
    assert (whole[:, n:] == 0).all()
