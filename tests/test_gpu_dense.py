"""The dense operators (dgsparse.embedding, rms_norm / add_rms_norm / add_rms_norm_fp8, gated_ffn, quantize_fp8 / matmul_fp8) against plain
implementations in 64 bits, at the sizes and masks where they can go wrong.

Tolerances are derived, element by element, from the arithmetic: U(t) = finfo(t).eps / 2 for a value rounded once to its type, n * 2^-24 * sum |terms|
for a sum of n terms held in 32 bits (whatever its order), and the propagation of an input's error through the formula."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
ids_of = lambda t: str(t).replace('torch.', '')  # noqa: E731
E32 = 2.0 ** -24


def U(t):
    return torch.finfo(t).eps / 2


def tiny(t):  # half a step below the smallest normal value
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def within(got, want, bound, what):
    got, want = got.double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= bound) & ~(got.isnan() & want.isnan())
    if bad.any():
        i = bad.nonzero()[0]
        b = torch.as_tensor(bound, device=got.device).expand_as(got)
        raise AssertionError(f'{what}: {int(bad.sum())} of {bad.numel()} beyond the bound; first at {i.tolist()}: {got[tuple(i)].item()!r}, '
                             f'want {want[tuple(i)].item()!r}, bound {b[tuple(i)].item():.3g}')


def rand(*shape, t, seed, scale=1.0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    return (torch.randn(*shape, generator=g, device='cuda') * scale).to(t)


# ---- embedding --------------------------------------------------------------------------------------------------------------
def embedding_want(ids, table, scale, dout, pad):
    """(out, dtable, sum of |terms|, terms) in 64 bits."""
    V, D = table.shape
    flat = ids.reshape(-1).long()
    ok = (flat >= 0) & (flat < V)
    out = torch.zeros(flat.numel(), D, dtype=torch.float64, device=table.device)
    out[ok] = table.double()[flat[ok]] * float(scale)
    out[flat >= V] = math.nan
    grad = ok & (flat != pad) if pad is not None else ok
    d = dout.reshape(-1, D).double()[grad]
    dtable = torch.zeros(V, D, dtype=torch.float64, device=table.device).index_add_(0, flat[grad], d * float(scale))
    mag = torch.zeros_like(dtable).index_add_(0, flat[grad], d.abs() * abs(float(scale)))
    cnt = torch.bincount(flat[grad], minlength=V).double()
    return out.view(*ids.shape, D), dtable, mag, cnt


def check_embedding(ids, table, scale=1.0, pad=None, seed=0, dout=None):
    import dgsparse
    t = table.dtype
    tab = table.detach().requires_grad_()
    out = dgsparse.embedding(ids, tab, scale=scale, padding_idx=pad)
    if dout is None:
        dout = rand(*out.shape, t=t, seed=seed + 1)
    dtable, = torch.autograd.grad(out, tab, dout)
    want, wtable, mag, cnt = embedding_want(ids, table, scale, dout, pad)
    # one product in 32 bits, one rounding
    within(out, want, want.abs() * (U(t) + 2 * E32) + tiny(t), 'out')
    # cnt additions and a product in 32 bits, one rounding
    within(dtable, wtable, wtable.abs() * U(t) + (cnt[:, None] + 2) * E32 * mag * (1 + U(t)) + tiny(t), 'dtable')
    assert torch.equal(out, dgsparse.embedding(ids, table, scale=scale)) or out.isnan().any()
    again, = torch.autograd.grad(dgsparse.embedding(ids, tab, scale=scale, padding_idx=pad), tab, dout)
    assert torch.equal(again.view(torch.uint8), dtable.view(torch.uint8)), 'the gradient differs between two runs'
    return out, dtable


@pytest.mark.parametrize('t', TYPES, ids=ids_of)
@pytest.mark.parametrize('n,V,D', [(1, 1, 1), (1, 7, 8), (2, 3, 5), (33, 50, 130), (64, 3, 1000), (31, 33, 4096), (257, 100, 24), (4096, 300, 16),
                                   (4097, 300, 16), (8192, 500, 8), (8193, 500, 8), (10000, 97, 40), (20000, 70000, 8), (9000, 1 << 19, 3), (9000, (1 << 20) + 7, 2), (3000, 129, 2056)])
def test_embedding_matches_64_bits(n, V, D, t):
    g = torch.Generator(device='cuda').manual_seed(n)
    ids = torch.randint(0, V, (n,), generator=g, device='cuda')
    check_embedding(ids, rand(V, D, t=t, seed=V), scale=0.5 if n % 2 else 3.0)


@pytest.mark.parametrize('t', TYPES, ids=ids_of)
def test_embedding_no_token_beyond_the_table_and_padding(t):
    ids = torch.tensor([[0, -1, 4, 2], [2, 2, 9, -7], [5, 1 << 40, 3, 2]], device='cuda')
    out, dtable = check_embedding(ids, rand(5, 12, t=t, seed=3), scale=2.0, pad=2)
    assert out[0, 1].eq(0).all() and out[1, 3].eq(0).all() and out[1, 2].isnan().all() and out[2, 0].isnan().all() and out[2, 1].isnan().all()
    assert dtable[2].eq(0).all() and dtable[1].eq(0).all() and dtable[0].ne(0).any()
    # not one token at all
    check_embedding(torch.full((70,), -1, device='cuda'), rand(5, 12, t=t, seed=3))
    check_embedding(torch.full((9000,), 5, device='cuda', dtype=torch.int32), rand(5, 12, t=t, seed=3))


@pytest.mark.parametrize('n', [65, 3000, 20000])
def test_embedding_one_token_at_every_place(n):
    """The row's sum crosses every chunk's border; its neighbours have none, or one at the list's ends."""
    ids = torch.full((n,), 3, device='cuda')
    check_embedding(ids, rand(6, 72, t=torch.float32, seed=1))
    ids[0], ids[-1] = 5, 0
    check_embedding(ids, rand(6, 72, t=torch.bfloat16, seed=1))


def test_embedding_runs_of_every_length_across_chunks():
    ids = torch.repeat_interleave(torch.arange(150, device='cuda'), torch.arange(150, device='cuda'))  # runs of 0 .. 149
    for perm in (False, True):
        if perm:
            ids = ids[torch.randperm(ids.numel(), device='cuda')]
        check_embedding(ids, rand(151, 20, t=torch.float32, seed=2))
        check_embedding(ids[:4000], rand(151, 20, t=torch.float16, seed=2))


def test_embedding_layouts():
    import dgsparse
    wide = rand(60, 96, t=torch.bfloat16, seed=5)
    table = wide[:, 8:72]  # rows of 64 in rows of 96, at 16-byte multiples
    ids = torch.randint(0, 60, (7, 11, 2), device='cuda')
    check_embedding(ids[..., 0], table)
    check_embedding(ids.int().transpose(0, 1), wide[:, 3:70])  # not at 16-byte multiples
    check_embedding(ids[..., 1], rand(64, 60, t=torch.float32, seed=4).t())  # columns
    # a broadcast gradient, and a transposed one
    check_embedding(ids[..., 0], table, dout=rand(1, 1, 64, t=torch.bfloat16, seed=6).expand(7, 11, 64))
    check_embedding(ids[:, 0, 0], table, dout=rand(64, 7, t=torch.bfloat16, seed=6).t())
    # nothing to look up
    empty = dgsparse.embedding(ids[:0], table.detach().requires_grad_())
    assert empty.shape == (0, 11, 2, 64)
    tab = table.detach().clone().requires_grad_()
    assert torch.autograd.grad(dgsparse.embedding(ids[:0], tab).sum(), tab)[0].eq(0).all()


def test_embedding_table_beyond_32_bits():
    V, D = 530000, 4096  # 2.17e9 values: element offsets pass 2^31
    table = torch.empty(V, D, dtype=torch.float16, device='cuda')
    ids = torch.tensor([V - 1, 0, V - 2, V - 1, 524287, 524289], device='cuda')
    rows = rand(6, D, t=torch.float16, seed=8)
    table[ids] = rows
    tab = table.requires_grad_()
    import dgsparse
    out = dgsparse.embedding(ids, tab)
    assert torch.equal(out, table.detach()[ids])
    dout = rand(6, D, t=torch.float16, seed=9)
    grad, = torch.autograd.grad(out, tab, dout)
    assert torch.equal(grad[0], dout[1]) and torch.equal(grad[524287], dout[4]) and torch.equal(grad[524289], dout[5]) and torch.equal(grad[V - 2], dout[2])
    assert torch.equal(grad[V - 1], (dout[0].float() + dout[3].float()).half())
    touched = torch.zeros(V, dtype=torch.bool, device='cuda')
    touched[ids] = True
    assert int((grad != 0).any(dim=1).ne(touched).sum()) == 0


# ---- RMS norm ---------------------------------------------------------------------------------------------------------------
NORM_SIZES = [(1, 1), (3, 5), (9, 64), (7, 128), (65, 129), (40, 256), (33, 1000), (6, 1024), (5, 2048), (5, 4096), (4, 8192), (3, 16384), (2, 16390), (2, 20000), (1500, 72)]


def norm_want(s, w, eps, dy, ds):
    v = s.double()
    r = (v.square().mean(-1, keepdim=True) + eps).rsqrt()
    wd = w.double()
    y = v * r * wd
    dyd = dy.double()
    dot = (v * wd * dyd).mean(-1, keepdim=True)
    dx = r * wd * dyd - v * r ** 3 * dot + (ds.double() if ds is not None else 0)
    # magnitudes that the roundings in 32 bits go with
    mag = (r * wd * dyd).abs() + v.abs() * r ** 3 * (v * wd * dyd).abs().mean(-1, keepdim=True) + (ds.double().abs() if ds is not None else 0)
    return y, dx, mag, (dyd * v * r).sum(0), (dyd * v * r).abs().sum(0)


@pytest.mark.parametrize('t', TYPES, ids=ids_of)
@pytest.mark.parametrize('rows,D', NORM_SIZES)
def test_add_rms_norm_matches_64_bits(rows, D, t):
    import dgsparse
    x, res = rand(rows, D, t=t, seed=1), rand(rows, D, t=t, seed=2, scale=3.0)
    w = (1 + rand(D, t=torch.float32, seed=3, scale=0.1)).to(t)
    dy, ds = rand(rows, D, t=t, seed=4), rand(rows, D, t=t, seed=5)
    leaves = [a.requires_grad_() for a in (x, res, w)]
    y, s = dgsparse.add_rms_norm(*leaves, eps=1e-5)
    assert torch.equal(s, (x.float() + res.float()).to(t)), 's is the sum, rounded once'
    dx, dres, dw = torch.autograd.grad((y, s), leaves, (dy, ds))
    wy, wdx, mag, wdw, wmag = norm_want(s.detach(), w.detach(), 1e-5, dy, ds)
    n = D + 16  # a mean over D, its root, and some products
    within(y, wy, wy.abs() * (U(t) + n * E32) + tiny(t), 'y')
    within(dx, wdx, wdx.abs() * U(t) + 2 * n * E32 * mag + tiny(t), 'dx')
    assert torch.equal(dx, dres)
    within(dw, wdw, wdw.abs() * U(t) + (n + rows) * E32 * wmag + tiny(t), 'dw')
    # the other forms: no residual; an output without a gradient; no gradient wanted
    sd = s.detach().clone().requires_grad_()
    y2 = dgsparse.rms_norm(sd, w, eps=1e-5)
    assert torch.equal(y2, y)
    dx2, dw2 = torch.autograd.grad(y2, (sd, w), dy)
    wy, wdx, mag, _, _ = norm_want(s.detach(), w.detach(), 1e-5, dy, None)
    within(dx2, wdx, wdx.abs() * U(t) + 2 * n * E32 * mag + tiny(t), 'dx without ds')
    assert torch.equal(dw2, dw)
    y3, s3 = dgsparse.add_rms_norm(*leaves, eps=1e-5)
    only, = torch.autograd.grad(s3, (x,), ds)
    assert torch.equal(only, ds)
    y4, s4 = dgsparse.add_rms_norm(*leaves, eps=1e-5)
    only, = torch.autograd.grad(y4, (x,), dy)
    assert torch.equal(only, dx2)
    with torch.no_grad():
        y5, s5 = dgsparse.add_rms_norm(x, res, w, eps=1e-5)
    assert torch.equal(y5, y) and torch.equal(s5, s) and not y5.requires_grad


def test_rms_norm_gradient_against_differences():
    import dgsparse
    x, w = rand(3, 40, t=torch.float32, seed=1).requires_grad_(), (1 + rand(40, t=torch.float32, seed=2, scale=0.2)).requires_grad_()
    dy = rand(3, 40, t=torch.float32, seed=3)
    dx, dw = torch.autograd.grad(dgsparse.rms_norm(x, w, 1e-3), (x, w), dy)
    f = lambda a, b: (a * (a.square().mean(-1, keepdim=True) + 1e-3).rsqrt() * b * dy.double()).sum()  # noqa: E731
    step = 2.0 ** -12
    for leaf, grad, pick in ((x, dx, 0), (w, dw, 1)):
        base = [x.detach().double(), w.detach().double()]
        flat = base[pick].view(-1)
        for i in range(0, flat.numel(), 17):
            old = flat[i].item()
            flat[i] = old + step
            hi = f(*base)
            flat[i] = old - step
            lo = f(*base)
            flat[i] = old
            # central difference: third derivative (order 10 here) * step^2 / 6; the gradient itself in 32 bits
            assert abs(((hi - lo) / (2 * step)).item() - grad.view(-1)[i].item()) < 1e-5 * (1 + abs(grad.view(-1)[i].item()))


def test_rms_norm_layouts_and_odd_values():
    import dgsparse
    w = rand(64, t=torch.float16, seed=1)
    big = rand(20, 160, t=torch.float16, seed=2)
    for x in (big[:, 16:80], big[:, 3:67], big[::2, 8:72], rand(64, 9, t=torch.float16, seed=3).t(), big[0, :64], big[:, :128].reshape(5, 4, 2, 64)[:, 1],
              rand(1, 64, t=torch.float16, seed=4).expand(6, 64)):
        c = x.contiguous()
        assert torch.equal(dgsparse.rms_norm(x, w), dgsparse.rms_norm(c, w))
        y, s = dgsparse.add_rms_norm(x, c, w)
        yc, sc = dgsparse.add_rms_norm(c, c, w)
        assert torch.equal(y, yc) and torch.equal(s, sc) and s.shape == x.shape
    # rows of zeros (eps alone), of infinities, of NaN; a row does not touch its neighbours
    x = rand(5, 64, t=torch.float16, seed=5)
    clean = dgsparse.rms_norm(x, w)
    x[1], x[3, 7] = 0, math.nan
    y = dgsparse.rms_norm(x, w)
    assert y[1].eq(0).all() and y[3].isnan().all() and torch.equal(y[[0, 2, 4]], clean[[0, 2, 4]])
    assert dgsparse.rms_norm(x[:0], w).shape == (0, 64)
    y, s = dgsparse.add_rms_norm(x[:0].requires_grad_(), x[:0], w.detach().requires_grad_())
    (y.sum() + s.sum()).backward()


def e4m3_step(q):
    """Half a step of e4m3 around |q|: 2^-4 relative, 2^-10 below the smallest normal value 2^-6."""
    return torch.clamp(q.abs() * 2.0 ** -4, min=2.0 ** -10)


@pytest.mark.parametrize('t', TYPES, ids=ids_of)
@pytest.mark.parametrize('rows,D', NORM_SIZES)
def test_add_rms_norm_fp8_matches_64_bits(rows, D, t):
    import dgsparse
    x, res = rand(rows, D, t=t, seed=1), rand(rows, D, t=t, seed=2, scale=3.0)
    w = (1 + rand(D, t=torch.float32, seed=3, scale=0.1)).to(t)
    q, scale, s = dgsparse.add_rms_norm_fp8(x.requires_grad_(), res, w, eps=1e-5)
    assert q.dtype == torch.float8_e4m3fn and scale.shape == (rows, -(-D // 128)) and not q.requires_grad
    assert torch.equal(s, (x.detach().float() + res.float()).to(t))
    v = s.double()
    y = v * (v.square().mean(-1, keepdim=True) + 1e-5).rsqrt() * w.double()
    n = (D + 16) * E32
    for b in range(scale.shape[1]):
        part = y[:, 128 * b:128 * b + 128]
        want = part.abs().amax(dim=1) / 448
        within(scale[:, b], want, want * (n + 2 * E32), 'scale')
        quot = part / scale[:, b].double()[:, None]
        within(q[:, 128 * b:128 * b + 128].float(), quot, e4m3_step(quot) * (1 + 2.0 ** -4) + quot.abs() * (n + 2 * E32), 'q')


def test_add_rms_norm_fp8_odd_values():
    import dgsparse
    w = torch.ones(300, device='cuda')
    x = rand(4, 300, t=torch.float32, seed=1)
    x[0], x[1, 140], x[2, 5] = 0, math.nan, math.inf
    q, scale, s = dgsparse.add_rms_norm_fp8(x, torch.zeros_like(x), w)
    assert q[0].float().eq(0).all() and scale[0].eq(2.0 ** -96 / 448).all()
    assert q[1].float().isnan().all() and scale[1].isnan().all()  # (the row's mean is NaN)
    assert q[2].float().isnan().any() and q[3].float().isfinite().all() and scale[3].isfinite().all()


# ---- gated feed-forward -----------------------------------------------------------------------------------------------------
def act64(name, g):
    if name == 'relu':
        return g.clamp_min(0), (g > 0).double()
    if name == 'silu':
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    c = 0.5 * torch.erfc(-g / math.sqrt(2))
    return g * c, c + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)


def ffn_want(x, wg, wu, dh, name):
    """{output: (value, bound)} in 64 bits.  t's operands are exact; sums of n products are off by n 2^-24 sum |terms|."""
    t = x.dtype
    X, G, W, H = x.double(), wg.double(), wu.double(), dh.double()
    D, F, T = X.shape[1], G.shape[0], X.shape[0]
    g, u = X @ G.t(), X @ W.t()
    eg, eu = D * E32 * (X.abs() @ G.abs().t()), D * E32 * (X.abs() @ W.abs().t())
    a, d = act64(name, g)
    # act and act' in 32 bits: exp's argument is rounded (|g| steps), some operations; |act'| <= 1.13, |act''| <= 0.8
    ulp = (g.abs() + 16) * 2 * E32
    ea = 1.13 * eg + ulp * a.abs() + 4 * E32 * g.abs()
    ed = (0.8 * eg if name != 'relu' else 0.0) + ulp * (d.abs() + 1)
    h = a * u
    eh = ea * (u.abs() + eu) + a.abs() * eu + h.abs() * (U(t) + 4 * E32) + tiny(t)
    dg, du = H * u * d, H * a
    edg = H.abs() * ((u.abs() + eu) * ed + eu * d.abs()) + dg.abs() * (U(t) + 4 * E32) + tiny(t)
    edu = H.abs() * ea + du.abs() * (U(t) + 4 * E32) + tiny(t)
    dx = dg @ G + du @ W
    edx = edg @ G.abs() + edu @ W.abs() + 2 * (F + 8) * E32 * ((dg.abs() + edg) @ G.abs() + (du.abs() + edu) @ W.abs()) + dx.abs() * U(t) + tiny(t)
    res = dict(h=(h, eh), dx=(dx, edx))
    for k, p, e in (('dw_gate', dg, edg), ('dw_up', du, edu)):
        v = p.t() @ X
        res[k] = (v, e.t() @ X.abs() + (T + 64) * E32 * ((p.abs() + e).t() @ X.abs()) + v.abs() * U(t) + tiny(t))
    return res


def check_ffn(x, wg, wu, name, seed=0, dh=None):
    import dgsparse
    leaves = [a.detach().requires_grad_() for a in (x, wg, wu)]
    h = dgsparse.gated_ffn(*leaves, activation=name)
    if dh is None:
        dh = rand(*h.shape, t=x.dtype, seed=seed + 9)
    dx, dwg, dwu = torch.autograd.grad(h, leaves, dh)
    D, F = x.shape[-1], wg.shape[0]
    want = ffn_want(x.detach().reshape(-1, D), wg.detach(), wu.detach(), dh.reshape(-1, F), name)
    for k, v in dict(h=h.reshape(-1, F), dx=dx.reshape(-1, D), dw_gate=dwg, dw_up=dwu).items():
        within(v, *want[k], what=k)
    # the projections kept, or made again: both ways on each case
    for again in (False, True):
        h2 = dgsparse.gated_ffn(*leaves, activation=name, recompute=again)
        for k, v in zip(('h', 'dx', 'dw_gate', 'dw_up'), (h2,) + torch.autograd.grad(h2, leaves, dh)):
            within(v.reshape(want[k][0].shape), *want[k], what=f'{k} recompute={again}')
    assert torch.equal(h, dgsparse.gated_ffn(x.detach(), wg.detach(), wu.detach(), name))
    return h, dx, dwg, dwu


FFN_SIZES = [(1, 1, 1), (1, 8, 16), (2, 5, 7), (3, 72, 40), (16, 256, 33), (17, 100, 33), (32, 40, 130), (64, 264, 128), (65, 64, 64), (66, 602, 10), (130, 136, 72), (129, 50, 300),
             (257, 512, 520), (1000, 96, 160), (5000, 64, 128)]


@pytest.mark.parametrize('t', TYPES, ids=ids_of)
@pytest.mark.parametrize('T,D,F', FFN_SIZES)
def test_gated_ffn_matches_64_bits(T, D, F, t):
    name = ('silu', 'gelu')[(T + D) % 2]
    check_ffn(rand(T, D, t=t, seed=1), rand(F, D, t=t, seed=2, scale=D ** -0.5), rand(F, D, t=t, seed=3, scale=D ** -0.5), name)


@pytest.mark.parametrize('t', TYPES, ids=ids_of)
@pytest.mark.parametrize('T,D,F', [(2049, 72, 2820), (300, 2000, 2100)])
def test_gated_ffn_large_tiles(T, D, F, t):
    """Enough tiles for the largest shape in the forward pass and in each product of the backward pass."""
    check_ffn(rand(T, D, t=t, seed=1), rand(F, D, t=t, seed=2, scale=D ** -0.5), rand(F, D, t=t, seed=3, scale=D ** -0.5), 'silu')


@pytest.mark.parametrize('t', TYPES, ids=ids_of)
@pytest.mark.parametrize('T', [5, 70])
def test_gated_ffn_relu_on_whole_numbers(T, t):
    """Whole numbers: every product is exact, so that both sides see the same sign, 0 among them."""
    g = torch.Generator(device='cuda').manual_seed(T)
    x, wg, wu = (torch.randint(-2, 3, s, generator=g, device='cuda').to(t) for s in ((T, 24), (40, 24), (40, 24)))
    check_ffn(x, wg, wu, 'relu', dh=torch.randint(-3, 4, (T, 40), generator=g, device='cuda').to(t))


def test_gated_ffn_layouts():
    t = torch.bfloat16
    wide = rand(90, 200, t=t, seed=1)
    wg, wu = rand(48, 64, t=t, seed=2, scale=0.1), rand(48, 64, t=t, seed=3, scale=0.1)
    both = rand(96, 64, t=t, seed=4, scale=0.1)
    check_ffn(wide[:, 8:72], wg, wu, 'silu')             # rows at a distance
    check_ffn(wide[:, 3:67], wg, wu, 'silu')             # not at 16-byte multiples
    check_ffn(wide[:64].t(), wg, wu, 'gelu')             # columns
    check_ffn(wide[:, :192].reshape(30, 3, 3, 64), both[:48], both[48:], 'silu')  # halves of one weight, x in more dimensions
    check_ffn(wide[0, :64], both[::2], both[1::2], 'silu')
    check_ffn(wide[:, :64], rand(48, 128, t=t, seed=4, scale=0.1)[:, :64], wu, 'silu')  # weights with different distances
    check_ffn(wide[:70, :64], wg, wu, 'silu', dh=rand(1, 48, t=t, seed=5).expand(70, 48))
    check_ffn(rand(1, 64, t=t, seed=5).expand(70, 64), wg, wu, 'silu')
    import dgsparse
    leaves = [wide[:0, :64].detach().requires_grad_(), wg.requires_grad_(), wu.requires_grad_()]
    h = dgsparse.gated_ffn(*leaves)
    assert h.shape == (0, 48)
    h.sum().backward()
    assert leaves[1].grad.eq(0).all() and leaves[2].grad.eq(0).all()


def test_gated_ffn_partial_gradients_and_odd_values():
    import dgsparse
    x, wg, wu = rand(80, 40, t=torch.float32, seed=1), rand(50, 40, t=torch.float32, seed=2, scale=0.2), rand(50, 40, t=torch.float32, seed=3, scale=0.2)
    h, dx, dwg, dwu = check_ffn(x, wg, wu, 'gelu')
    dh = rand(80, 50, t=torch.float32, seed=9)
    a = x.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(dgsparse.gated_ffn(a, wg, wu, 'gelu'), a, dh)[0], dx)
    b = wu.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(dgsparse.gated_ffn(x, wg, b, 'gelu'), b, dh)[0], dwu)
    # an infinity or a NaN stays in its row; tails read as zeros, never as a neighbour's values
    bad = x.clone()
    bad[7, 3], bad[79, 39] = math.nan, math.inf
    hb = dgsparse.gated_ffn(bad, wg, wu, 'silu')
    good = torch.ones(80, dtype=torch.bool, device='cuda')
    good[[7, 79]] = False
    assert hb[7].isnan().all() and not hb[79].isfinite().all() and torch.equal(hb[good], dgsparse.gated_ffn(x, wg, wu, 'silu')[good])
    # large arguments: silu'(-200) = 0, not NaN
    big = torch.full((70, 8), 100.0, device='cuda', requires_grad=True)
    w = torch.full((8, 8), -1.0, device='cuda')
    out = dgsparse.gated_ffn(big, w, w, 'silu')
    assert out.isfinite().all() and torch.autograd.grad(out.sum(), big)[0].isfinite().all()


# ---- 8 bits -----------------------------------------------------------------------------------------------------------------
def dequantized(q, scale, rows):
    s = scale.double().repeat_interleave(rows, 0)[:q.shape[0]].repeat_interleave(128, 1)[:, :q.shape[1]]
    return q.float().double() * s


@pytest.mark.parametrize('t', TYPES, ids=ids_of)
@pytest.mark.parametrize('rows,cols', [(1, 1), (3, 5), (7, 128), (130, 129), (128, 256), (300, 1000), (257, 640)])
@pytest.mark.parametrize('block_rows', [1, 128])
def test_quantize_fp8(rows, cols, block_rows, t):
    import dgsparse
    x = rand(rows, cols, t=t, seed=rows)
    x[rows // 2] = 0
    q, scale = dgsparse.quantize_fp8(x, block_rows)
    assert scale.shape == (-(-rows // block_rows), -(-cols // 128))
    for i in range(scale.shape[0]):
        for j in range(scale.shape[1]):
            part = x[i * block_rows:(i + 1) * block_rows, 128 * j:128 * j + 128].double()
            want = part.abs().max().clamp_min(2.0 ** -96) / 448
            within(scale[i, j], want, want * E32, 'scale')
            quot = part / scale[i, j].double()
            within(q[i * block_rows:(i + 1) * block_rows, 128 * j:128 * j + 128].float(), quot, e4m3_step(quot) * (1 + 2.0 ** -4) + quot.abs() * E32, 'q')
    wide = rand(rows, cols + 9, t=t, seed=2)
    for v in (wide[:, 3:3 + cols], wide[:, 8:8 + cols]):
        a, b = dgsparse.quantize_fp8(v, block_rows), dgsparse.quantize_fp8(v.contiguous(), block_rows)
        assert torch.equal(a[0].view(torch.uint8), b[0].view(torch.uint8)) and torch.equal(a[1], b[1])


def check_mm8(a, sa, b, sb, t):
    import dgsparse
    out = dgsparse.matmul_fp8(a, sa, b, sb, t)
    A, B = dequantized(a.reshape(-1, a.shape[-1]), sa.reshape(-1, sa.shape[-1]), 1), dequantized(b, sb, 128)
    want, mag = A @ B.t(), A.abs() @ B.abs().t()
    K = b.shape[1]
    # K products, a scale's product and an addition for each block in 32 bits
    within(out.reshape(want.shape), want, (K + 4 * (-(-K // 128)) + 8) * E32 * mag + want.abs() * U(t) + tiny(t), 'out')
    return out


MM8_SIZES = [(1, 1, 1), (1, 16, 128), (5, 40, 128), (16, 130, 304), (17, 16, 1040), (33, 64, 256), (64, 300, 1000), (65, 129, 129), (200, 500, 384), (300, 1000, 1040), (70, 60, 4096), (2049, 6001, 272)]


@pytest.mark.parametrize('t', TYPES, ids=ids_of)
@pytest.mark.parametrize('M,N,K', MM8_SIZES)
def test_matmul_fp8_matches_64_bits(M, N, K, t):
    import dgsparse
    a, sa = dgsparse.quantize_fp8(rand(M, K, t=torch.float32, seed=1))
    # rows and blocks of very different size: a wrong scale shows
    w = rand(N, K, t=torch.float32, seed=2) * (1 + torch.arange(N, device='cuda')[:, None] // 128) / (1 + torch.arange(K, device='cuda') // 128)
    b, sb = dgsparse.quantize_fp8(w, 128)
    sa = sa * torch.linspace(0.5, 2, sa.numel(), device='cuda').view_as(sa)
    check_mm8(a, sa, b, sb, t)


def test_matmul_fp8_layouts():
    import dgsparse
    a, sa = dgsparse.quantize_fp8(rand(6, 5, 256, t=torch.float32, seed=1))
    b, sb = dgsparse.quantize_fp8(rand(70, 256, t=torch.float32, seed=2), 128)
    out = check_mm8(a, sa, b, sb, torch.float16)
    assert out.shape == (6, 5, 70)
    wide = torch.empty(30, 300, dtype=torch.uint8, device='cuda')
    for at in (16, 3):
        v = wide[:, at:at + 256].view(torch.float8_e4m3fn) if at == 16 else wide.view(torch.float8_e4m3fn)[:, at:at + 256]
        v.view(torch.uint8).copy_(a.reshape(30, 256).view(torch.uint8))
        assert torch.equal(dgsparse.matmul_fp8(v, sa.reshape(30, 2), b, sb, torch.float16), out.reshape(30, 70))
    assert torch.equal(dgsparse.matmul_fp8(a[0], sa.transpose(0, 1).contiguous().transpose(0, 1)[0], b, sb, torch.float16), out[0])
    assert dgsparse.matmul_fp8(a[:0], sa[:0], b, sb).shape == (0, 5, 70)
    # a NaN stays in its row
    n = a.clone().view(torch.uint8)
    n[2, 1, 200] = 0x7f
    bad = dgsparse.matmul_fp8(n.view(torch.float8_e4m3fn), sa, b, sb, torch.float16)
    assert bad[2, 1].isnan().all() and torch.equal(bad[:2], out[:2]) and torch.equal(bad[3:], out[3:])


# ---- where few rows end -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('t', TYPES, ids=ids_of)
@pytest.mark.parametrize('T,D,F', [(33, 72, 40), (48, 264, 130), (49, 40, 64), (64, 136, 5119), (49, 24, 5200), (64, 40, 5200)])
def test_gated_ffn_on_either_side_of_few_rows(T, D, F, t):
    check_ffn(rand(T, D, t=t, seed=1), rand(F, D, t=t, seed=2, scale=D ** -0.5), rand(F, D, t=t, seed=3, scale=D ** -0.5), 'gelu')


@pytest.mark.parametrize('t', TYPES, ids=ids_of)
@pytest.mark.parametrize('M,N,K', [(16, 4100, 4200), (17, 4100, 4200), (32, 4096, 4096), (32, 4112, 4096), (33, 40, 300), (17, 1, 4096)])
def test_matmul_fp8_on_either_side_of_few_rows(M, N, K, t):
    import dgsparse
    a, sa = dgsparse.quantize_fp8(rand(M, K, t=torch.float32, seed=1))
    b, sb = dgsparse.quantize_fp8(rand(N, K, t=torch.float32, seed=2), 128)
    check_mm8(a, sa, b, sb, t)


def test_gated_ffn_rows_of_infinities_in_the_tiles():
    """32 bits beyond the few rows: an infinity is a NaN in the rows that it reaches, and in no other."""
    import dgsparse
    x, wg, wu = rand(200, 40, t=torch.float32, seed=1), rand(70, 40, t=torch.float32, seed=2, scale=0.2), rand(70, 40, t=torch.float32, seed=3, scale=0.2)
    bad = x.clone()
    bad[[0, 63, 128, 199], [0, 3, 39, 17]] = torch.tensor([math.inf, -math.inf, math.inf, -math.inf], device='cuda')
    h = dgsparse.gated_ffn(bad, wg, wu, 'gelu')
    good = torch.ones(200, dtype=torch.bool, device='cuda')
    good[[0, 63, 128, 199]] = False
    assert h[~good].isnan().all() and torch.equal(h[good], dgsparse.gated_ffn(x, wg, wu, 'gelu')[good])


# ---- together, streams, graphs ----------------------------------------------------------------------------------------------
def chain(ids, table, norm, wg, wu, aq, asc):
    """lookup -> residual norm -> gated product -> 8-bit projection"""
    import dgsparse
    x = dgsparse.embedding(ids, table, scale=4.0)
    y, s = dgsparse.add_rms_norm(x, x, norm)
    h = dgsparse.gated_ffn(y, wg, wu, 'silu')
    q, qs = dgsparse.quantize_fp8(h)
    n8, n8s, _ = dgsparse.add_rms_norm_fp8(y, s, norm)
    return h, s, dgsparse.matmul_fp8(q, qs, aq, asc, torch.float32), n8, n8s


def chain_inputs(seed, t=torch.bfloat16):
    import dgsparse
    g = torch.Generator(device='cuda').manual_seed(seed)
    ids = torch.randint(-1, 500, (5000,), generator=g, device='cuda')
    w = [rand(500, 64, t=t, seed=seed), 1 + rand(64, t=t, seed=seed + 1, scale=0.1), rand(96, 64, t=t, seed=seed + 2, scale=0.1), rand(96, 64, t=t, seed=seed + 3, scale=0.1)]
    return ids, w, dgsparse.quantize_fp8(rand(48, 96, t=torch.float32, seed=seed + 4), 128)


def test_run_of_all_captured_and_replayed():
    """Forward and backward of the run in one graph, replayed with new inputs between the program's own eager work; two graphs with their own workspaces."""
    ids, w, (aq, asc) = chain_inputs(1)
    static_ids, dh = ids.clone(), rand(5000, 96, t=torch.bfloat16, seed=7)
    leaves = [a.detach().clone().requires_grad_() for a in w]

    def step():
        h, s, o, n8, n8s = chain(static_ids, *leaves, aq, asc)
        return (h.detach(), o, n8s) + torch.autograd.grad((h, s), leaves, (dh, torch.ones_like(s)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for k in range(4):
        static_ids.copy_(chain_inputs(10 + k)[0])
        eager = [v.clone() for v in step()]
        torch.cuda.synchronize()
        for graph, out in graphs if k % 2 else graphs[::-1]:
            graph.replay()
        torch.cuda.synchronize()
        for graph, out in graphs:
            for a, b in zip(out, eager):
                assert torch.equal(a, b), k


def test_run_on_two_streams_at_once():
    work = [chain_inputs(20 + k) for k in range(2)]
    want = [[v.clone() for v in chain(ids, *w, aq, asc)] for ids, w, (aq, asc) in work]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(5):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                ids, w, (aq, asc) = work[k]
                got[k] = chain(ids, *w, aq, asc)
        torch.cuda.synchronize()
        for k in range(2):
            for a, b in zip(got[k], want[k]):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_gradient_of_a_gradient_is_refused():
    import dgsparse
    x, w = rand(70, 16, t=torch.float32, seed=1).requires_grad_(), rand(8, 16, t=torch.float32, seed=2).requires_grad_()
    for f in (lambda: dgsparse.gated_ffn(x, w, w), lambda: dgsparse.rms_norm(x, w[0]), lambda: dgsparse.embedding(torch.zeros(3, dtype=torch.int, device='cuda'), x)):
        with pytest.raises(RuntimeError, match='differentiable once'):
            torch.autograd.grad(f().sum(), x, create_graph=True)
    assert torch.autograd.grad(dgsparse.gated_ffn(x, w, w).sum(), w)[0].shape == w.shape
