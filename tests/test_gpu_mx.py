"""GPU: activation checkpoints in 8 bits and 4-bit weights (csrc/mx8.hip, csrc/mx4.hip) against float64.

Codes, scales and restored values are whole numbers times powers of two and have to be EQUAL.  Computed results carry bounds formed
per element from the float64 terms: a rounding is half a step (2^-24 relative in fp32, 2^-8 in bf16), a step of the matrix
pipe's accumulator one step (2^-23, it truncates)."""
import pytest
import torch

import mx_forms
import mx_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def dev():
    assert torch.cuda.is_available(), 'gpu tests need a GPU'
    return torch.device('cuda:0')


@pytest.fixture
def x3_mode():
    from iprgan import _lib
    before = _lib.get_math()
    _lib.set_math('fp32x3')
    yield
    _lib.set_math(before)


def rnd(*shape, seed=0, scale=1.0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale


def same(a, b):
    """Equal, NaN where NaN."""
    a, b = a.detach().cpu().double(), b.detach().cpu().double()
    return a.shape == b.shape and bool(((a == b) | (torch.isnan(a) & torch.isnan(b))).all())


def awkward(n, seed):
    """Values over the whole exponent range, zero blocks, block maxima on both sides of the rounding borders, subnormals."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, generator=g) * torch.exp2(torch.randint(-140, 126, (n,), generator=g).float().clamp(-126, 126))
    x = torch.where(torch.rand(n, generator=g) < 0.1, torch.zeros(n), x)
    b = torch.arange(n) // 32
    scale = torch.exp2((torch.randint(-100, 100, (int(b[-1]) + 1,), generator=g)).float())[b]
    y = torch.randn(n, generator=g) * scale
    x = torch.where(b % 3 == 0, x, y)
    x = torch.where(b % 7 == 5, torch.zeros(n), x)
    # whole multiples of half a step under a block maximum of exactly 1: ties
    t = torch.randint(-255, 256, (n,), generator=g).float() / 128
    x = torch.where(b % 5 == 2, t, x)
    t4 = torch.randint(-28, 29, (n,), generator=g).float() / 4
    x = torch.where(b % 5 == 4, t4, x)
    lim = torch.tensor([127.5 / 64, 127.49 / 64, 1.0, 1.75, 1.7499999, 2.0, 7.0, 6.9999995, 3.3e38, 3.4e38, 1e-45, 1e-38, 2.0 ** -128])
    k = min(n // 32, len(lim))
    for j in range(k):
        x[32 * j] = lim[j]
        x[32 * j + 1:32 * j + 32] = x[32 * j + 1:32 * j + 32].clamp(-1e-3 * lim[j], 1e-3 * lim[j]) if j % 2 else 0
    return x


# ---- 8-bit checkpoints ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('n', [1, 3, 8, 31, 32, 33, 100, 1000, 4096, 40001])
@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_mx8_codes_and_values(dev, n, dtype):
    from iprgan import ops
    x = awkward(n, n)
    x = x if dtype == 'f32' else x.bfloat16()
    q = ops.mx8_quant(x.to(dev))
    codes, scales = R.mx8_encode(x)
    assert torch.equal(q.scales.cpu(), scales)
    assert torch.equal(q.codes.cpu(), codes)
    back = ops.mx8_dequant(q)
    assert back.dtype == x.dtype and back.shape == x.shape
    assert same(back, R.mx8_decode(codes, scales))
    f = ops.mx8_dequant(q, ops.ST_F32)
    assert same(f, R.mx8_decode(codes, scales))
    # at most half a step away, a whole one where the exponent cap saturates
    sc = scales.repeat_interleave(32)[:n]
    step = torch.exp2(sc.double() - 127)
    err = (f.cpu().double() - x.double()).abs()
    assert bool(((err <= torch.where(sc == 248, step, step / 2)) | (sc == 255)).all())


def test_mx8_three_planes(dev, x3_mode):
    from iprgan import ops
    for shape in ((3, 5, 7, 64), (2, 3, 3, 36)):
        x = rnd(*shape, seed=3)
        t = ops.to_kind(x.to(dev), ops.ST_X3)
        q = ops.mx8_quant(t)
        codes, scales = R.mx8_encode(x)
        assert q.kind == ops.ST_X3 and torch.equal(q.codes.cpu(), codes) and torch.equal(q.scales.cpu(), scales)
        back = ops.mx8_dequant(q)
        assert ops.is16(back) == ops.ST_X3
        assert torch.equal(ops.f32(back).cpu().double().view(-1), R.mx8_decode(codes, scales))
        part = ops.mx8_quant(t[1:])                   # a batch slice keeps its parent's plane stride
        codes, scales = R.mx8_encode(x[1:])
        assert torch.equal(part.codes.cpu(), codes) and torch.equal(part.scales.cpu(), scales)


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_mx8_views_off_a_16_byte_boundary(dev, dtype):
    from iprgan import ops
    flat = rnd(4 * 4 * 12 + 6, seed=8)
    flat = (flat if dtype == 'f32' else flat.bfloat16()).to(dev)
    stats = rnd(1 + 4 * 12, seed=9).abs().add(0.5).to(dev)
    for off in (1, 2, 4):
        v = flat[off:off + 192].view(1, 4, 4, 12)
        q, r = ops.mx8_quant(v), ops.mx8_quant(v.clone())
        assert torch.equal(q.codes, r.codes) and torch.equal(q.scales, r.scales)
        p = [stats[1 + 12 * i:13 + 12 * i] for i in range(4)]
        a = ops.bn_bwd(q, None, v, p[0], p[1], p[2], 1, beta=p[3])
        b = ops.bn_bwd(q, None, v.clone(), p[0].clone(), p[1].clone(), p[2].clone(), 1, beta=p[3].clone())
        assert all(torch.equal(s, t) for s, t in zip(a, b))
        assert torch.equal(ops.act_bwd(v, q, 1), ops.act_bwd(v.clone(), q, 1))


def test_mx8_non_finite_blocks_read_back_as_nan(dev):
    from iprgan import ops
    x = rnd(32 * 6 + 5, seed=1)
    x[3], x[70], x[101], x[-1] = float('nan'), float('inf'), float('-inf'), float('inf')
    got = ops.mx8_dequant(ops.mx8_quant(x.to(dev))).cpu()
    bad = torch.zeros(x.numel(), dtype=torch.bool)
    for b in (0, 2, 3, 6):
        bad[32 * b:32 * b + 32] = True
    assert bool(torch.isnan(got[bad]).all()) and bool(torch.isfinite(got[~bad]).all())


NORMS = [
    # form, shape, act, affine
    ('bn', (4, 9, 7, 64), 1, True), ('bn', (4, 9, 7, 64), 2, True), ('bn', (4, 9, 7, 64), 0, True),
    ('bn', (3, 5, 5, 36), 2, True), ('bn', (2, 3, 3, 4), 1, True), ('bn', (1, 1, 17, 260), 1, True), ('bn', (2, 4, 4, 1024), 2, True),
    ('bn', (16, 33, 31, 20), 1, True), ('bn', (64, 32, 32, 8), 2, True),
    ('inst', (4, 9, 7, 64), 1, True), ('inst', (4, 9, 7, 64), 2, False), ('inst', (70, 4, 5, 12), 1, True), ('inst', (3, 64, 64, 32), 0, True),
    ('inst', (1, 17, 1, 516), 2, True), ('inst', (2, 1, 1, 8), 1, True),
    ('prelu', (4, 9, 7, 64), 2, True), ('prelu', (3, 6, 5, 36), 2, True), ('prelu', (16, 24, 24, 64), 2, True),
]


def norm_inputs(form, shape, affine, seed=0):
    b, h, w, c = shape
    G = b if form == 'inst' else 1
    M = b * h * w // G
    x = rnd(*shape, seed=seed) * torch.exp(0.3 * rnd(c, seed=seed + 1)) + rnd(c, seed=seed + 2)
    codes, scales = R.mx8_encode(x)
    xg = x.view(G, M, c)
    mean = xg.mean(1)
    invstd = 1 / torch.sqrt(xg.var(1, unbiased=False) + 1e-5)
    gamma = (1 + 0.3 * rnd(c, seed=seed + 3)) if affine else None
    if affine:
        gamma[0] = -gamma[0].abs()                     # a flipped sign (the mask's comparison turns round) and a zero scale
        gamma[1] = 0.0
    beta = 0.3 * rnd(c, seed=seed + 4) if affine else None
    dy = rnd(*shape, seed=seed + 5)
    return G, M, codes, scales, mean, invstd, gamma, beta, dy


def norm_reference(G, M, c, codes, scales, mean, invstd, gamma, beta, dy, act, slope):
    """float64 results and, for each, the bound of an fp32 evaluation: every operation half a step, a sum of M terms taken in
    chains of at most D additions (rows a thread walks + row lanes + partial rows: below 300 here) D + 8 half steps."""
    x = R.mx8_decode(codes, scales).view(G, M, c)
    g = dy.double().view(G, M, c)
    m, i = mean.double().view(G, 1, c), invstd.double().view(G, 1, c)
    ga = gamma.double() if gamma is not None else torch.ones(c, dtype=torch.float64)
    be = beta.double() if beta is not None else torch.zeros(c, dtype=torch.float64)
    t = (x - m) * i
    v = t * ga + be
    dz = g if act == 0 else torch.where(v > 0, g, g * (slope if act == 2 else 0.0))
    s1, s2 = dz.sum(1, keepdim=True), (dz * t).sum(1, keepdim=True)
    k = ga * i
    dx = k * (dz - s1 / M - t * s2 / M)
    u, D = 2.0 ** -24, 300
    a1, a2 = dz.abs().sum(1, keepdim=True), (dz * t).abs().sum(1, keepdim=True)
    tdx = k.abs() * u * (6 * dz.abs() + (D + 8) * a1 / M + (D + 12) * t.abs() * a2 / M) + 1e-37
    ds = (g * v.clamp(max=0)).sum()
    tds = u * (D + 16) * (g.abs() * (t * ga).abs() + g.abs() * be.abs()).sum()
    return dict(dx=dx, tdx=tdx, dg=s2.sum(0).view(c), tdg=(u * (D + 16) * a2.sum(0)).view(c) + 1e-37, db=s1.sum(0).view(c),
                tdb=(u * (D + 16) * a1.sum(0)).view(c) + 1e-37, ds=ds, tds=tds)


def run_norm(form, q, dy, gamma, mean, invstd, act, slope, beta, dev, **kw):
    from iprgan import ops
    to = lambda t: None if t is None else t.to(dev)
    if form == 'prelu':
        return ops.bn_prelu_bwd(q, dy, to(gamma), to(beta), to(mean), to(invstd), torch.full((1,), slope, device=dev), **kw)
    f = ops.bn_bwd if form == 'bn' else ops.instnorm_bwd
    return f(q, None, dy, to(gamma), to(mean), to(invstd), act, slope, beta=to(beta), **kw)


@pytest.mark.parametrize('form,shape,act,affine', NORMS)
@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_norm_backward_from_the_checkpoint(dev, form, shape, act, affine, dtype):
    from iprgan import ops
    c = shape[-1]
    G, M, codes, scales, mean, invstd, gamma, beta, dy = norm_inputs(form, shape, affine)
    slope = {0: 0.0, 1: 0.0, 2: 0.25}[act]
    dy = dy if dtype == 'f32' else dy.bfloat16()
    ref = norm_reference(G, M, c, codes, scales, mean, invstd, gamma, beta, dy, act, slope)
    q = ops.Mx8(codes.to(dev), scales.to(dev), shape)
    dbias = torch.full((c,), 2.0, device=dev)
    out = run_norm(form, q, dy.to(dev), gamma, mean, invstd, act, slope, beta, dev, dbias=dbias, dbias_beta=0.5)
    dx = out[0].cpu().double().view(G, M, c)
    assert out[0].dtype == dy.dtype and tuple(out[0].shape) == shape
    tdx = ref['tdx'] + (2.0 ** -8 * ref['dx'].abs() if dtype == 'bf16' else 0)
    assert bool(((dx - ref['dx']).abs() <= tdx).all()), float(((dx - ref['dx']).abs() / tdx).max())
    if affine:
        assert bool(((out[1].cpu().double() - ref['dg']).abs() <= ref['tdg']).all())
        assert bool(((out[2].cpu().double() - ref['db']).abs() <= ref['tdb']).all())
    else:
        assert out[1] is None and out[2] is None
    if form == 'prelu':
        assert abs(float(out[3].cpu()) - float(ref['ds'])) <= float(ref['tds'])
    # the column sums of dx, accumulated onto half of what was there: each dx within its bound, the sum in chains as above
    want = 1.0 + ref['dx'].sum((0, 1))
    tol = ref['tdx'].sum((0, 1)) + 2.0 ** -24 * 400 * (ref['dx'].abs().sum((0, 1)) + 2)
    assert bool(((dbias.cpu().double() - want).abs() <= tol).all())
    again = run_norm(form, q, dy.to(dev), gamma, mean, invstd, act, slope, beta, dev)
    assert all(a is None or torch.equal(a, b) for a, b in zip(out, again)), 'not deterministic'


def test_norm_backward_mask_is_exact_next_to_zero(dev):
    """Inputs that ARE the threshold: v = 0 exactly counts as not positive, one code further as positive."""
    from iprgan import ops
    c = 8
    codes = torch.zeros(64 * c, dtype=torch.int8)
    codes.view(64, c)[:] = torch.arange(-32, 32)[:, None]
    scales = torch.full((64 * c // 32,), 127, dtype=torch.uint8)            # step 1: the values are the codes
    mean = torch.full((1, c), 3.0)
    invstd = torch.full((1, c), 0.3)
    gamma = torch.tensor([1.0, -1.0, 0.7, -0.7, 1e-3, 0.0, 0.0, 5.0])
    beta = torch.tensor([0.0, 0.0, 0.0, 0.0, 0.0, 1e-30, -1e-30, 0.0])
    dy = torch.ones(1, 8, 8, c)
    q = ops.Mx8(codes.to(dev), scales.to(dev), (1, 8, 8, c))
    _, _, db = ops.bn_bwd(q, None, dy.to(dev), gamma.to(dev), mean.view(c).to(dev), invstd.view(c).to(dev), 1, beta=beta.to(dev))
    pos = torch.arange(-32, 32)[:, None].double() - 3
    want = torch.where(gamma.double() == 0, beta.double().expand(64, c) > 0, pos * gamma.double().sign() > 0).double().sum(0)
    assert torch.equal(db.cpu().double(), want)


@pytest.mark.parametrize('rows', [1 << 9, 1 << 19])
def test_slope_gradient_keeps_its_precision(dev, rows):
    """The PReLU slope's gradient is one sum over the whole tensor.  Here the second half of the rows repeats the first with the opposite
    gradient, all but one row, so that it is far smaller than its parts.  It is taken in 64 bits; a block's sum is stored as two floats
    (2^-48 of it off), their totals and the result are rounded to one: 3 half steps of the result, 16 allowed; 64-bit sums in
    chains shorter than 2^12 are off by 2^-41 of the terms' absolute sum, and 2^-40 is allowed."""
    from iprgan import ops
    c, half = 64, rows // 2
    g = torch.Generator(device=dev).manual_seed(5)
    x = torch.randn(half, c, generator=g, device=dev)
    dy = torch.rand(half, c, generator=g, device=dev) + 0.5
    q = ops.mx8_quant(torch.cat([x, x]).view(1, rows // 256, 256, c))
    dy = torch.cat([dy, -dy])
    dy[-1] = 1e-3
    dy = dy.view(1, rows // 256, 256, c)
    gamma, beta = torch.rand(c, generator=g, device=dev) + 0.5, torch.randn(c, generator=g, device=dev)
    mean, invstd = 0.1 * torch.randn(c, generator=g, device=dev), torch.rand(c, generator=g, device=dev) + 0.5
    got = ops.bn_prelu_bwd(q, dy, gamma, beta, mean, invstd, torch.full((1,), 0.25, device=dev))[3]
    v = (ops.mx8_dequant(q).double() - mean.double()) * invstd.double() * gamma.double() + beta.double()
    t = v.clamp(max=0) * dy.double()
    assert abs(float(got) - float(t.sum())) <= 2.0 ** -20 * abs(float(t.sum())) + 2.0 ** -40 * float(t.abs().sum())


def test_norm_backward_three_planes(dev, x3_mode):
    """fp32x3: three-plane dy -> three-plane dx; an fp32 dy next to a checkpoint of a splitting layer -> three-plane dx."""
    from iprgan import ops
    shape, c = (4, 9, 7, 64), 64
    G, M, codes, scales, mean, invstd, gamma, beta, dy = norm_inputs('bn', shape, True)
    ref = norm_reference(G, M, c, codes, scales, mean, invstd, gamma, beta, dy, 2, 0.2)
    for kx, kd in ((ops.ST_F32, ops.ST_F32), (ops.ST_X3, ops.ST_X3), (ops.ST_F32, ops.ST_X3)):
        q = ops.Mx8(codes.to(dev), scales.to(dev), shape, kx)
        d = ops.to_kind(dy.to(dev), kd)
        dx, dg, db = ops.bn_bwd(q, None, d, gamma.to(dev), mean.view(c).to(dev), invstd.view(c).to(dev), 2, 0.2, beta=beta.to(dev))
        assert ops.is16(dx) == ops.ST_X3
        err = (ops.f32(dx).cpu().double().view(G, M, c) - ref['dx']).abs()
        assert bool((err <= ref['tdx'] * 1.01).all())
        assert bool(((dg.cpu().double() - ref['dg']).abs() <= ref['tdg']).all())


@pytest.mark.parametrize('n', [1, 7, 32, 1000, 4099])
@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_act_backward_from_the_checkpoint(dev, n, dtype):
    from iprgan import ops
    out = torch.tanh(rnd(n, seed=n))
    dy = rnd(n, seed=n + 1)
    dy = dy if dtype == 'f32' else dy.bfloat16()
    codes, scales = R.mx8_encode(out)
    o = R.mx8_decode(codes, scales)
    q = ops.Mx8(codes.to(dev), scales.to(dev), (n,))
    for act, slope in ((0, 0.0), (1, 0.0), (2, 0.2), (3, 0.0), (4, 0.0)):
        got = ops.act_bwd(dy.to(dev), q, act, slope).cpu().double()
        s32 = float(torch.tensor(slope))                          # the slope as the fp32 it is handed over as
        d = {0: torch.ones_like(o), 1: (o > 0).double(), 2: torch.where(o > 0, 1.0, s32).double(), 3: 1 - o * o,
             4: (1 + o) * (1 - o) / 2}[act]
        want = dy.double() * d
        # 1 - o^2 cancels: its absolute error is a few half steps of one
        tol = dy.double().abs() * 4 * 2.0 ** -24 + (2.0 ** -8 * want.abs() if dtype == 'bf16' else 0)
        assert bool(((got - want).abs() <= tol).all())


# ---- 4-bit weights -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('rows,cols', [(1, 1), (3, 7), (5, 27), (2, 32), (7, 100), (4, 128), (3, 129), (64, 576), (17, 1000), (9, 4104)])
@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_mx4_codes_and_values(dev, rows, cols, dtype):
    from iprgan import ops
    x = awkward(rows * cols, rows * cols).view(rows, cols)
    x = x if dtype == 'f32' else x.bfloat16()
    q = ops.mx4_quant(x.to(dev))
    codes, scales = R.mx4_encode(x)
    assert torch.equal(q.scales.cpu(), scales)
    want = R.mx4_decode(codes, scales, cols)
    assert same(R.mx4_decode(q.codes, q.scales, cols), want)
    c = q.codes.cpu()
    nib = torch.stack([c & 15, c >> 4], 2).view(rows, -1)
    assert bool((nib[:, cols:] & 7 == 0).all()), 'padding must be zero codes'
    assert same(ops.mx4_dequant(q), want)
    assert same(ops.mx4_dequant(q, torch.bfloat16), want)


def test_mx4_non_finite_blocks(dev):
    from iprgan import ops
    x = rnd(4, 160, seed=1)
    x[1, 40], x[2, 0], x[3, 159] = float('nan'), float('inf'), float('-inf')
    v = ops.mx4_dequant(ops.mx4_quant(x.to(dev))).cpu()
    bad = torch.zeros(4, 160, dtype=torch.bool)
    bad[1, 32:64] = bad[2, :32] = bad[3, 128:] = True
    assert bool(torch.isnan(v[bad]).all()) and bool(torch.isfinite(v[~bad]).all())
    # ... and so do the products
    y = ops.mx4_linear(rnd(3, 160, seed=2).to(dev), ops.mx4_quant(x.to(dev))).cpu()
    assert bool(torch.isnan(y[:, 1:]).all()) and bool(torch.isfinite(y[:, 0]).all())
    y = ops.mx4_linear(ops.mx4_quant(rnd(3, 160, seed=2).to(dev)), ops.mx4_quant(x.to(dev))).cpu()
    assert bool(torch.isnan(y[:, 1:]).all()) and bool(torch.isfinite(y[:, 0]).all())
    d = ops.mx4_linear_bwd(rnd(3, 4, seed=3).to(dev), ops.mx4_quant(x.to(dev))).cpu()
    badk = bad.any(0)
    assert bool(torch.isnan(d[:, badk]).all()) and bool(torch.isfinite(d[:, ~badk]).all())


LINEAR = [(1, 128, 64), (1, 16, 5), (2, 100, 33), (3, 27, 1), (16, 128, 256), (17, 130, 70), (31, 64, 129), (33, 513, 65), (64, 1152, 96),
          (65, 200, 130), (129, 384, 260), (100, 2000, 40), (5, 20000, 7), (300, 96, 300), (1, 1, 1), (130, 640, 514)]


def lin_bound(xa, wa, K, planes):
    """Half a step an accumulation (one step on the matrix pipe): K / 32 instructions a plane, the adds across splits and the epilogue."""
    return 2.0 ** -23 * (planes * (K // 32 + 1) + 72) * (xa @ wa) + 1e-37


@pytest.mark.parametrize('M,K,N', LINEAR)
@pytest.mark.parametrize('kind', ['f32', 'bf16', 'mx4'])
def test_mx4_linear(dev, M, K, N, kind):
    from iprgan import ops
    x, w = rnd(M, K, seed=1), rnd(N, K, seed=2) / K ** 0.5
    wc, wsc = R.mx4_encode(w)
    w4 = ops.Mx4(wc.to(dev), wsc.to(dev), (N, K))
    wd = R.mx4_decode(wc, wsc, K).t()
    if kind == 'bf16':
        x = x.bfloat16()
    xin = x.to(dev)
    xd = x.double()
    if kind == 'mx4':
        xin = ops.mx4_quant(xin)
        xd = R.mx4_decode(*R.mx4_encode(x), K)
    bias = rnd(N, seed=3)
    for act, slope, b, dt in ((0, 0.0, None, None), (1, 0.0, bias, None), (2, 0.2, bias, torch.bfloat16), (3, 0.0, None, torch.float32), (4, 0.0, bias, torch.float32)):
        y = ops.mx4_linear(xin, w4, None if b is None else b.to(dev), act, slope, dtype=dt)
        assert y.dtype == (dt or (torch.float32 if kind == 'mx4' else x.dtype)) and tuple(y.shape) == (M, N)
        pre = xd @ wd + (b.double() if b is not None else 0)
        want = R.act(pre, act, float(torch.tensor(slope)))
        tol = lin_bound(xd.abs(), wd.abs(), K, 3 if kind == 'f32' else 1) + 2.0 ** -24 * pre.abs() * 2
        tol = tol + 4 * 2.0 ** -24 * want.abs() + (2.0 ** -22 if act >= 3 else 0)          # the activation's own evaluation
        tol = tol + (2.0 ** -8 * want.abs() if y.dtype == torch.bfloat16 else 0)
        err = (y.cpu().double() - want).abs()
        assert bool((err <= tol).all()), (act, float((err / tol).max()))
    assert torch.equal(y, ops.mx4_linear(xin, w4, bias.to(dev), 4, 0.0, dtype=torch.float32)), 'not deterministic'


@pytest.mark.parametrize('M,K,N', LINEAR)
@pytest.mark.parametrize('kind', ['f32', 'bf16'])
def test_mx4_linear_backward(dev, M, K, N, kind):
    from iprgan import ops
    dy, w = rnd(M, N, seed=1), rnd(N, K, seed=2)
    wc, wsc = R.mx4_encode(w)
    w4 = ops.Mx4(wc.to(dev), wsc.to(dev), (N, K))
    wd = R.mx4_decode(wc, wsc, K)
    dy = dy if kind == 'f32' else dy.bfloat16()
    for dt in (None, torch.float32, torch.bfloat16):
        dx = ops.mx4_linear_bwd(dy.to(dev), w4, dtype=dt)
        want = dy.double() @ wd
        tol = lin_bound(dy.double().abs(), wd.abs(), N, 3 if kind == 'f32' else 1)
        tol = tol + (2.0 ** -8 * want.abs() if dx.dtype == torch.bfloat16 else 0)
        assert dx.dtype == (dt or dy.dtype) and tuple(dx.shape) == (M, K)
        err = (dx.cpu().double() - want).abs()
        assert bool((err <= tol).all()), float((err / tol).max())


def test_mx4_linear_gradient_against_differences(dev):
    """y is linear in x: a central difference along any direction is the gradient's product with it, up to the roundings of y."""
    from iprgan import ops
    M, K, N = 6, 96, 80
    w4 = ops.mx4_quant(rnd(N, K, seed=2).to(dev))
    x, d, dy = rnd(M, K, seed=1), rnd(M, K, seed=4), rnd(M, N, seed=3)
    up, dn = ops.mx4_linear((x + d).to(dev), w4), ops.mx4_linear((x - d).to(dev), w4)
    num = (((up - dn).cpu().double() / 2) * dy.double()).sum()
    ana = (ops.mx4_linear_bwd(dy.to(dev), w4).cpu().double() * d.double()).sum()
    scale = ((x.abs() + d.abs()).double() @ ops.mx4_dequant(w4).cpu().double().abs().t() * dy.abs().double()).sum()
    assert abs(float(num - ana)) <= 2.0 ** -23 * 100 * float(scale)


@pytest.mark.parametrize('M,K,N', [(1000, 1024, 700), (2304, 2048, 5888), (100, 20000, 70), (70, 33000, 200), (257, 128, 300), (129, 256, 40)])
def test_mx4_product_stages_and_splits(dev, M, K, N):
    """Both operands in 4 bits: K in whole and odd numbers of stages, split over blocks, one tile and several a block, repeated (float64 on
    the device)."""
    from iprgan import ops
    xq = ops.mx4_quant(rnd(M, K, seed=1).to(dev))
    wq = ops.mx4_quant((rnd(N, K, seed=2) / K ** 0.5).to(dev))
    bias = rnd(N, seed=3).to(dev)
    xd, wd = ops.mx4_dequant(xq).double(), ops.mx4_dequant(wq).double().t().contiguous()
    want = xd @ wd + bias.double()
    tol = lin_bound(xd.abs(), wd.abs(), K, 1) + 2.0 ** -23 * want.abs()
    first = ops.mx4_linear(xq, wq, bias, dtype=torch.float32)
    err = (first.double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
    for _ in range(3):
        assert torch.equal(first, ops.mx4_linear(xq, wq, bias, dtype=torch.float32))


@pytest.mark.parametrize('M,K,N', [(4099, 300, 3101), (2304, 1700, 5888)])
def test_mx4_product_of_many_rows(dev, M, K, N):
    """More tiles than the chip runs at once, ragged edges, both operands in 4 bits (float64 on the device)."""
    from iprgan import ops
    x, w = rnd(M, K, seed=1).to(dev), rnd(N, K, seed=2).to(dev) / K ** 0.5
    xq, wq = ops.mx4_quant(x), ops.mx4_quant(w)
    y = ops.mx4_linear(xq, wq, dtype=torch.float32).double()
    xd, wd = ops.mx4_dequant(xq).double(), ops.mx4_dequant(wq).double().t().contiguous()
    err, tol = (y - xd @ wd).abs(), lin_bound(xd.abs(), wd.abs(), K, 1)
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize('M,K,N', [(2050, 130, 4100), (2050, 77, 4099), (40, 515, 16001), (70, 6000, 1025), (200, 4100, 2049), (300, 4096, 2047), (520, 2050, 640)])
@pytest.mark.parametrize('kind', ['f32', 'bf16'])
def test_mx4_linear_and_gradient_large_tiles(dev, M, K, N, kind):
    """Sizes that reach the tiles of many rows and columns, with rows of odd lengths, and views that start between two 4-byte words
    (float64 on the device)."""
    from iprgan import ops
    t = torch.float32 if kind == 'f32' else torch.bfloat16
    pl = 3 if kind == 'f32' else 1
    x, dy = rnd(M * K + 1, seed=1).to(dev, t), rnd(M * N + 1, seed=3).to(dev, t)
    w4 = ops.mx4_quant(rnd(N, K, seed=2).to(dev))
    wd = ops.mx4_dequant(w4).double()
    for o in (0, 1):
        a, d = x[o: o + M * K].view(M, K), dy[o: o + M * N].view(M, N)
        y, want = ops.mx4_linear(a, w4, dtype=torch.float32).double(), a.double() @ wd.t().contiguous()
        err, tol = (y - want).abs(), lin_bound(a.double().abs(), wd.abs().t().contiguous(), K, pl)
        assert bool((err <= tol).all()), float((err / tol).max())
        dx, want = ops.mx4_linear_bwd(d, w4, dtype=torch.float32).double(), d.double() @ wd
        err, tol = (dx - want).abs(), lin_bound(d.double().abs(), wd.abs(), N, pl)
        assert bool((err <= tol).all()), float((err / tol).max())


def test_mx4_linear_leading_dimensions_and_unaligned_views(dev):
    from iprgan import ops
    w4 = ops.mx4_quant(rnd(24, 64, seed=2).to(dev))
    x = rnd(2, 3, 5, 64, seed=1)
    y = ops.mx4_linear(x.to(dev), w4)
    assert tuple(y.shape) == (2, 3, 5, 24)
    assert torch.equal(y.view(30, 24), ops.mx4_linear(x.view(30, 64).to(dev), w4))
    assert tuple(ops.mx4_linear(x[0, 0, 0].to(dev), w4).shape) == (24,)
    flat = rnd(30 * 64 + 1, seed=5).to(dev)
    v = flat[1:].view(30, 64)                     # contiguous, 4-byte aligned only
    assert torch.equal(ops.mx4_linear(v, w4), ops.mx4_linear(v.clone(), w4))
    assert torch.equal(ops.mx4_quant(v).codes, ops.mx4_quant(v.clone()).codes)
    dflat = rnd(30 * 24 + 1, seed=6).to(dev)[1:].view(30, 24)
    assert torch.equal(ops.mx4_linear_bwd(dflat, w4), ops.mx4_linear_bwd(dflat.clone(), w4))
    b = torch.zeros(25, device=dev).normal_()[1:]
    assert torch.equal(ops.mx4_linear(v, w4, b), ops.mx4_linear(v, w4, b.clone()))


# ---- together, as a training step and a server use them -------------------------------------------------------------------
def test_operators_under_capture_and_on_another_stream(dev):
    """Quantise, restore, norm backward, quantised product and its gradient captured into one graph, replayed on new inputs with eager
    work between the replays; and run on a side stream: equal to the eager results each time."""
    from iprgan import ops
    shape, c = (4, 8, 8, 64), 64
    mean, invstd = (0.1 * rnd(c, seed=1)).to(dev), (1 + 0.1 * rnd(c, seed=2).abs()).to(dev)
    gamma, beta = rnd(c, seed=3).to(dev), rnd(c, seed=4).to(dev)
    w4 = ops.mx4_quant(rnd(96, c, seed=5).to(dev))
    x, dy = rnd(*shape, seed=6).to(dev), rnd(*shape, seed=7).to(dev)

    def work():
        q = ops.mx8_quant(x)
        dx, dg, db = ops.bn_bwd(q, None, dy, gamma, mean, invstd, 1, beta=beta)
        y = ops.mx4_linear(ops.mx8_dequant(q), w4, None, 2, 0.2)
        z = ops.mx4_linear(ops.mx4_quant(dx.view(-1, c)), w4)
        return [dx, dg, db, y, z, ops.mx4_linear_bwd(y.view(-1, 96), w4)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = work()
    for seed in (20, 21, 22):
        x.copy_(rnd(*shape, seed=seed))
        dy.copy_(rnd(*shape, seed=seed + 50))
        g.replay()
        torch.cuda.synchronize()
        eager = work()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager))
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = work()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(other, eager))


# ---- offsets past 32 bits (about 25 GB at a time; all but the ends of each tensor is zero) ------------------------------------------
def test_checkpoint_past_32_bits(dev):
    """2^32 + 4 113 elements: the end of the tensor is quantised and restored as it is by itself; a restore in fp32 passes 2^34 bytes."""
    from iprgan import ops
    n, k = (1 << 32) + 4113, 4096 + 17
    end = awkward(k, 5).bfloat16().to(dev)
    x = torch.zeros(n, dtype=torch.bfloat16, device=dev)
    x[-k:] = end
    q, own = ops.mx8_quant(x), ops.mx8_quant(end)
    assert torch.equal(q.codes[-k:], own.codes) and torch.equal(q.scales[(n - k) // 32:], own.scales)
    assert int(q.codes[:n - k].count_nonzero()) == 0
    del x
    for kind in (ops.ST_BF16, ops.ST_F32):
        y = ops.mx8_dequant(q, kind)
        assert same(y[-k:], ops.mx8_dequant(own, kind))
        assert int(y[:n - k].count_nonzero()) == 0
        del y
    dy = torch.zeros(n, dtype=torch.bfloat16, device=dev)
    dy[-k:] = rnd(k, seed=6).bfloat16()
    dz = ops.act_bwd(dy, q, 2, 0.25)
    assert same(dz[-k:], ops.act_bwd(dy[-k:].clone(), own, 2, 0.25))


def test_norm_backward_past_32_bits(dev):
    """2^26 + 5 rows of 64 channels; only the first and the last 1000 rows have gradients.  Sums: 2000 additions that are not of a zero, each off by
    at most half a step of the sum of the magnitudes, and 8 roundings a term; dx: 8 fp32 roundings of its terms and one to bf16."""
    from iprgan import ops
    M, C, k = (1 << 26) + 5, 64, 1000
    x = torch.zeros(M, C, dtype=torch.bfloat16, device=dev)
    dy = torch.zeros(M, C, dtype=torch.bfloat16, device=dev)
    for s, rows in ((1, slice(0, k)), (2, slice(M - k, M))):
        x[rows] = rnd(k, C, seed=s).bfloat16().to(dev)
        dy[rows] = rnd(k, C, seed=s + 10).bfloat16().to(dev)
    mean, invstd = 0.1 * rnd(C, seed=3), 1 + 0.1 * rnd(C, seed=4).abs()
    gamma, beta = rnd(C, seed=5), rnd(C, seed=6)
    ends = [ops.mx8_dequant(ops.mx8_quant(t.clone())).double().cpu() for t in (x[:k], x[M - k:])]
    q = ops.mx8_quant(x)
    g = torch.cat([dy[:k], dy[M - k:]]).double().cpu()
    del x
    dx, dgamma, dbeta = ops.bn_bwd(q, None, dy, gamma.to(dev), mean.to(dev), invstd.to(dev), 1, beta=beta.to(dev))
    t = (torch.cat(ends) - mean.double()) * invstd.double()
    dz = torch.where(t * gamma.double() + beta.double() > 0, g, 0.0)
    u = 2.0 ** -24
    for got, terms in ((dbeta, dz), (dgamma, dz * t)):
        mag = terms.abs().sum(0) + (dz.abs() * (mean * invstd).abs().double()).sum(0)
        assert bool(((got.cpu().double() - terms.sum(0)).abs() <= 2008 * u * mag).all())
    gi = gamma.double() * invstd.double()
    s1, s2 = dbeta.cpu().double() / M, dgamma.cpu().double() / M
    want = gi * (dz - s1 - t * s2)
    bound = want.abs() * 2.0 ** -8 + 16 * u * gi.abs() * (dz.abs() + s1.abs() + (t.abs() + (mean * invstd).abs().double()) * s2.abs())
    got = torch.cat([dx[:k], dx[M - k:]]).cpu().double()
    assert bool(((got - want).abs() <= bound).all())


def test_weights_past_32_bits(dev):
    """65 600 x 65 536 weights (2.15 GB of codes), whole numbers small enough that every product and sum is exact."""
    from iprgan import ops
    N, K, k = 65600, 65536, 5
    gen = torch.Generator().manual_seed(3)
    end = torch.tensor([0., 1, 2, 3, 4, 6, -1, -2, -6])[torch.randint(0, 9, (k, K), generator=gen)]
    end[:, ::32] = 6.                                            # (block maximum 6: scale 1, values are codes)
    x = torch.zeros(N, K, dtype=torch.bfloat16, device=dev)
    x[-k:] = end.to(dev)
    w = ops.mx4_quant(x)
    del x
    back = ops.mx4_dequant(w, torch.bfloat16)
    assert torch.equal(back[-k:].float().cpu(), end) and int(back[:N - k].count_nonzero()) == 0
    del back
    for M in (2, 70):
        xs = torch.randint(-2, 3, (M, K), generator=gen).float()
        xs[:, ::32] = 0.
        want = xs.double() @ end.double().t()
        assert float((xs.abs().double() @ end.abs().double().t()).max()) < 2 ** 24
        for a in (xs.to(dev), xs.bfloat16().to(dev), ops.mx4_quant(xs.to(dev))):
            y = ops.mx4_linear(a, w, dtype=torch.float32)
            assert torch.equal(y[:, -k:].double().cpu(), want) and int(y[:, :N - k].count_nonzero()) == 0
        dy = torch.zeros(M, N)
        dy[:, -k:] = torch.randint(-8, 9, (M, k), generator=gen).float()
        for d in (dy.to(dev), dy.bfloat16().to(dev)):
            assert torch.equal(ops.mx4_linear_bwd(d, w, torch.float32).double().cpu(), dy[:, -k:].double() @ end.double())


def test_results_past_32_bits(dev):
    """40 000 x 65 600 results (2.6e9) of short whole-number sums, the product's and the gradient's."""
    from iprgan import ops
    M, N, K = 40000, 65600, 96
    gen = torch.Generator().manual_seed(4)
    x = torch.randint(-2, 3, (M, K), generator=gen).float().to(dev)
    wt = torch.randint(-2, 3, (N, K), generator=gen).float()
    wt[:, ::32] = 6.
    w = ops.mx4_quant(wt.to(dev))
    rows = torch.tensor([0, 16384, 32735, 32736, M - 1])         # (row 32 736 passes 2^31 elements)
    xq = x.clone()
    xq[:, ::32] = 6.
    for a, src in ((x, x), (x.bfloat16(), x), (ops.mx4_quant(xq), xq)):
        y = ops.mx4_linear(a, w, dtype=torch.bfloat16)
        want = (src.cpu()[rows].double() @ wt.double().t()).bfloat16()
        assert torch.equal(y[rows.to(dev)].cpu(), want)
        del y
    wb = torch.randint(-2, 3, (K, N), generator=gen).float()
    wb[:, ::32] = 6.
    w = ops.mx4_quant(wb.to(dev))
    for d in (x, x.bfloat16()):
        dx = ops.mx4_linear_bwd(d, w, torch.bfloat16)
        assert torch.equal(dx[rows.to(dev)].cpu(), (x.cpu()[rows].double() @ wb.double()).bfloat16())
        del dx


@pytest.mark.parametrize('M', [(1 << 20) + 5, 256 * 128 * 128 + 1])
def test_more_than_a_million_rows(dev, M):
    """Every position of a batch of maps as a row: whole numbers small enough that products and sums are exact."""
    from iprgan import ops
    K, N = 32, 12
    gen = torch.Generator().manual_seed(4)
    wt = torch.randint(-2, 3, (N, K), generator=gen).float()
    wt[:, 0] = 6.                                                # (scale 1: the values are the codes)
    w = ops.mx4_quant(wt.to(dev))
    x = torch.randint(-2, 3, (M, K), generator=gen).float().to(dev)
    x[:, 0] = 6.
    want = torch.zeros(M, N, device=dev)
    for k in range(K):
        want += x[:, k:k + 1] * wt[:, k].to(dev)
    for a in (x, x.bfloat16(), ops.mx4_quant(x)):
        assert torch.equal(ops.mx4_linear(a, w, dtype=torch.float32), want)
    got = ops.mx4_linear(x, w, act=3)
    assert torch.equal(got[-70:], ops.mx4_linear(x[-70:].clone(), w, act=3))
    dy = torch.randint(-8, 9, (M, N), generator=gen).float().to(dev)
    want = torch.zeros(M, K, device=dev)
    for n in range(N):
        want += dy[:, n:n + 1] * wt[n].to(dev)
    for d in (dy, dy.bfloat16()):
        assert torch.equal(ops.mx4_linear_bwd(d, w, torch.float32), want)


@pytest.mark.parametrize('form,G,M,C', [('inst', 1024, 1 << 17, 4), ('inst', 64, 4096, 4096), ('bn', 1, 1 << 20, 2048)])
@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_norm_sums_of_long_runs_of_rows(dev, form, G, M, C, dtype):
    """Tensors of which one thread walks 256 to 1024 rows or more.  A large gradient in the first rows and ones behind it: an fp32 sum that
    is not handed on to a wider one in time drops every one of them (a thousand of them: 2^-14 of the sum).  A sum in 64 bits of fp32 sums of
    256 rows is off by 256 half steps of the magnitudes, by 4 more for the stored partial sums and the result; every term here is exact.  The
    column sums of dx: gamma = invstd = 1, s1 / M and s2 / M the rounded sums, 8 roundings a dx, 256 + 4 of the sum."""
    from iprgan import ops
    n = G * M * C
    codes = torch.full((n,), 1, dtype=torch.int8, device=dev)
    scales = torch.full((n // 32,), 127, dtype=torch.uint8, device=dev)
    dy = torch.ones(G, M, 1, C, dtype=torch.float32 if dtype == 'f32' else torch.bfloat16, device=dev)
    dy[:, :256] = 2.0 ** 24
    mean, inv, gamma, beta = torch.zeros(G, C, device=dev), torch.ones(G, C, device=dev), torch.ones(C, device=dev), torch.ones(C, device=dev)
    q = ops.Mx8(codes, scales, dy.shape)
    db = torch.zeros(C, device=dev)
    f = (lambda *a, **k: ops.bn_bwd(*a[:4], a[4].view(C), a[5].view(C), *a[6:], **k)) if form == 'bn' else ops.instnorm_bwd
    dx, dgamma, dbeta = f(q, None, dy, gamma, mean, inv, 1, beta=beta, dbias=db)
    one = 256 * 2.0 ** 24 + (M - 256)                                      # a group's sum; x = 1: both sums are the same
    u = 2.0 ** -24
    for got in (dgamma, dbeta):
        assert float((got.double() - G * one).abs().max()) <= (256 + 4) * u * G * one
    s = torch.tensor(one).float().double()
    want = dx.double().sum((0, 1, 2)) if dtype == 'f32' else None
    if want is not None:                                                    # (bf16: dx is rounded again behind the sum)
        mag = dx.double().abs().sum((0, 1, 2))
        assert bool(((db.double() - want).abs() <= (256 + 4) * u * mag).all())
    big, rest = (2.0 ** 24 - 2 * float(s) / M), (1 - 2 * float(s) / M)
    tol = u * 264 * (2.0 ** 24 + 2 * float(s) / M) + (2.0 ** -8 * 2.0 ** 24 if dtype == 'bf16' else 0)
    assert float((dx[:, :256].double() - big).abs().max()) <= tol
    tol = u * 264 * (1 + 2 * float(s) / M) + (2.0 ** -8 * abs(rest) if dtype == 'bf16' else 0)
    assert float((dx[:, 256:].double() - rest).abs().max()) <= tol


@pytest.mark.parametrize('kind,n', [(k, n) for k in ('f32', 'bf16') for n in (1, 31, 32, 33, 1000, 40001)] + [('x3', 32), ('x3', 1000), ('x3', 40004)])
def test_mx8_signs(dev, kind, n, request):
    """Codes, scales and values as stated; value > 0 exactly where x > 0; act_bwd's mask is that of x."""
    from iprgan import ops
    x = awkward(n, n)
    x[n // 2] = 1e-45                                            # the smallest subnormal beside whatever its block holds
    if kind == 'x3':
        request.getfixturevalue('x3_mode')
        x = (rnd(n, seed=n) * torch.exp2(-8 * rnd(n, seed=n + 1).abs())).clamp(-4, 4)
        t = ops.to_kind(x.to(dev), ops.ST_X3)
    else:
        x = x if kind == 'f32' else x.bfloat16()
        t = x.to(dev)
    q = ops.mx8_quant(t, signs=True)
    codes, scales = R.mx8_encode_signs(x)
    assert torch.equal(q.scales.cpu(), scales) and torch.equal(q.codes.cpu(), codes)
    f = ops.mx8_dequant(q, ops.ST_F32).cpu()
    assert same(f, R.mx8_decode(codes, scales))
    fine = scales.repeat_interleave(32)[:n] != 255
    assert torch.equal((f > 0)[fine], (x > 0)[fine])
    back = ops.mx8_dequant(q)
    assert torch.equal((ops.f32(back) > 0).cpu()[fine], (x > 0)[fine])
    dy = rnd(n, seed=3)
    dz = ops.act_bwd(dy.to(dev), q, 1).cpu()
    assert torch.equal(dz[fine], torch.where(x > 0, dy, torch.zeros(n))[fine])


@pytest.mark.parametrize('kind,size,form', mx_forms.PRODUCT)
def test_every_form_of_the_product(dev, kind, size, form):
    """bias, LeakyReLU and both result types; K and N odd, the last rows and columns of a tile empty (float64 on the device)."""
    from iprgan import ops
    M, K, N = size
    g = torch.Generator(device=dev).manual_seed(7)
    x = torch.randn(M, K, generator=g, device=dev).to(torch.bfloat16 if kind == 'bf16' else torch.float32)
    w4 = ops.mx4_quant(torch.randn(N, K, generator=g, device=dev) / K ** 0.5)
    bias = torch.randn(N, generator=g, device=dev)
    xin = ops.mx4_quant(x) if kind == 'mx4' else x
    xd = ops.mx4_dequant(xin).double() if kind == 'mx4' else x.double()
    wd = ops.mx4_dequant(w4).double().t().contiguous()
    pre = xd @ wd + bias.double()
    want = torch.where(pre > 0, pre, pre * float(torch.tensor(0.2)))
    tol = lin_bound(xd.abs(), wd.abs(), K, 3 if kind == 'f32' else 1) + 4 * 2.0 ** -24 * pre.abs()
    for dt in (torch.float32, torch.bfloat16):
        y = ops.mx4_linear(xin, w4, bias, 2, 0.2, dtype=dt)
        err = (y.double() - want).abs()
        t = tol + (2.0 ** -8 * want.abs() if dt == torch.bfloat16 else 0)
        assert bool((err <= t).all()), (form, dt, float((err / t).max()))
        assert torch.equal(y, ops.mx4_linear(xin, w4, bias, 2, 0.2, dtype=dt)), 'not deterministic'


@pytest.mark.parametrize('kind,size,form', mx_forms.GRADIENT)
def test_every_form_of_the_gradient(dev, kind, size, form):
    from iprgan import ops
    M, K, N = size
    g = torch.Generator(device=dev).manual_seed(8)
    dy = torch.randn(M, N, generator=g, device=dev).to(torch.bfloat16 if kind == 'bf16' else torch.float32)
    w4 = ops.mx4_quant(torch.randn(N, K, generator=g, device=dev))
    wd = ops.mx4_dequant(w4).double()
    want, tol = dy.double() @ wd, lin_bound(dy.double().abs(), wd.abs(), N, 3 if kind == 'f32' else 1)
    for dt in (torch.float32, torch.bfloat16):
        dx = ops.mx4_linear_bwd(dy, w4, dtype=dt)
        err = (dx.double() - want).abs()
        t = tol + (2.0 ** -8 * want.abs() if dt == torch.bfloat16 else 0)
        assert bool((err <= t).all()), (form, dt, float((err / t).max()))
        assert torch.equal(dx, ops.mx4_linear_bwd(dy, w4, dtype=dt)), 'not deterministic'


@pytest.mark.parametrize('form,shape,affine', [(f, s, a) for f, s, a in [
    ('bn', (4, 9, 7, 64), True), ('bn', (3, 5, 5, 36), True), ('bn', (2, 3, 3, 4), True), ('bn', (1, 1, 17, 260), True), ('bn', (2, 4, 4, 1024), True),
    ('bn', (16, 33, 31, 20), True), ('inst', (4, 9, 7, 64), True), ('inst', (4, 9, 7, 64), False), ('inst', (70, 4, 5, 12), True),
    ('inst', (1, 17, 1, 516), True), ('inst', (2, 1, 1, 8), True), ('inst', (600, 5, 5, 132), False), ('bn', (9, 129, 129, 128), True)]])
@pytest.mark.parametrize('kind', ['f32', 'bf16', 'x3'])
def test_norm_inputs_keep_their_masks(dev, form, shape, affine, kind, request):
    """Codes and scales as stated; the mask read off the codes is that of x, counted by a gradient of ones (whole numbers: exact); nothing is off by a
    step or more.  The last shapes are walked in several strides, over several groups a stride."""
    from iprgan import ops
    if kind == 'x3':
        request.getfixturevalue('x3_mode')
    b, h, w, c = shape
    G = b if form == 'inst' else 1
    M = b * h * w // G
    x = rnd(*shape, seed=1) * torch.exp(0.3 * rnd(c, seed=2)) + rnd(c, seed=3)
    x = x.bfloat16() if kind == 'bf16' else x
    xg = x.float().view(G, M, c)
    mean, invstd = xg.mean(1), 1 / torch.sqrt(xg.var(1, unbiased=False) + 1e-5)
    gamma = (1 + 0.3 * rnd(c, seed=4)) if affine else None
    if affine:
        gamma[0], gamma[1] = -gamma[0].abs(), 0.0
    beta = 0.3 * rnd(c, seed=5) if affine else None
    codes, scales, mask = R.mx8_encode_norm(xg, gamma, beta, mean, invstd)
    to = lambda t: None if t is None else t.to(dev)
    t = ops.to_kind(x.to(dev), ops.ST_X3) if kind == 'x3' else x.to(dev)
    q = ops.mx8_quant(t, norm=(to(gamma), to(beta), to(mean if form == 'inst' else mean.view(c)), to(invstd if form == 'inst' else invstd.view(c))))
    assert torch.equal(q.scales.cpu(), scales) and torch.equal(q.codes.cpu(), codes)
    val = R.mx8_decode(codes, scales).view(xg.shape)
    step = torch.exp2(scales.double() - 127).repeat_interleave(32)[:codes.numel()].view(xg.shape)
    assert bool(((val - xg.double()).abs() < step).all())
    edge = codes.view(xg.shape).abs() == 127                     # (its neighbour on the other side would be 128: may have stayed)
    k = (gamma if affine else torch.ones(c)).double() * invstd.double().view(G, 1, c)
    got = (val - mean.double().view(G, 1, c)) * k + (beta if affine else torch.zeros(c)).double() > 0
    assert torch.equal(got[~edge], mask[~edge])
    if affine:
        f = ops.bn_bwd if form == 'bn' else ops.instnorm_bwd
        ms = [to(mean), to(invstd)] if form == 'inst' else [to(mean.view(c)), to(invstd.view(c))]
        db = f(q, None, torch.ones(shape, device=dev), to(gamma), *ms, 1, beta=to(beta))[2]
        assert torch.equal(db.cpu().double(), got.double().sum((0, 1)))


def test_norm_input_masks_refuse_what_does_not_fit(dev):
    from iprgan import ops
    x, v = torch.zeros(2, 3, 3, 8, device=dev), torch.ones(8, device=dev)
    for bad in ((v[:4], v[:4], v, v), (v, v, v[:4], v), (v, v, v, torch.ones(16, device=dev)), (v, v, torch.ones(40, device=dev), torch.ones(40, device=dev)),
                (v, None, v, v)):
        with pytest.raises(RuntimeError, match='mx8_quant'):
            ops.mx8_quant(x, norm=bad)
    with pytest.raises(RuntimeError, match='not both'):
        ops.mx8_quant(x, signs=True, norm=(v, v, v, v))
    with pytest.raises(RuntimeError, match='one device'):
        ops.mx8_quant(x, norm=(v.cpu(), v.cpu(), v, v))


def test_norm_input_masks_past_32_bits(dev):
    """2^32 + 512 elements and more in groups of 2^31 and of 128 channels: the end of the tensor as it is by itself."""
    from iprgan import ops
    C, M, G = 128, (1 << 24) + 4, 2
    tail = 40
    x = torch.zeros(G, M, 1, C, dtype=torch.bfloat16, device=dev)
    end = rnd(tail, C, seed=1).bfloat16().to(dev)
    x[1, -tail:, 0] = end
    mean, inv = 0.1 * rnd(G, C, seed=2).to(dev), 1 + 0.1 * rnd(G, C, seed=3).abs().to(dev)
    gamma, beta = rnd(C, seed=4).to(dev), 0.3 * rnd(C, seed=5).to(dev)
    q = ops.mx8_quant(x, norm=(gamma, beta, mean, inv))
    own = ops.mx8_quant(end.view(1, tail, 1, C), norm=(gamma, beta, mean[1:], inv[1:]))
    assert torch.equal(q.codes[-tail * C:], own.codes) and torch.equal(q.scales[-tail * C // 32:], own.scales)
    assert bool((q.scales[:-tail * C // 32] == 0).all())
