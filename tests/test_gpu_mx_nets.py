"""GPU: 8-bit checkpoints inside the chain executor (`engine: {ckpt8: true}`) and 4-bit dense layers of a served generator."""
import numpy as np
import pytest
import torch
import torch.nn as nn

import mx_reference as R
from oracle import cases, recipe

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def dev():
    assert torch.cuda.is_available(), 'gpu tests need a GPU'
    return torch.device('cuda:0')


@pytest.fixture
def ckpt8(monkeypatch):
    from iprgan import engine
    monkeypatch.setattr(engine, '_CKPT8_MIN', 1)

    def switch(on):
        monkeypatch.setattr(engine, '_CKPT8', on)
    yield switch


@pytest.fixture
def math(request):
    from iprgan import _lib
    before = _lib.get_math()
    _lib.set_math(request.param)
    yield request.param
    _lib.set_math(before)


def round8(t):
    """float64 NCHW tensor rounded as its NHWC (channels padded to 4) checkpoint is"""
    b, c, h, w = t.shape
    p = torch.zeros(b, h, w, (c + 3) & ~3, dtype=torch.float64)
    p[..., :c] = t.permute(0, 2, 3, 1)
    v = R.mx8_decode(*R.mx8_encode(p.float())).view(p.shape)
    return v[..., :c].permute(0, 3, 1, 2).contiguous()


def test_chain_gradients_are_those_of_the_rounded_activations(dev, ckpt8):
    """conv + LeakyReLU -> conv -> BatchNorm + ReLU -> conv, backward written out in float64 with every saved activation rounded to its
    checkpoint.  An activation that two evaluations of the forward pass round to neighbouring codes moves one term of a sum over
    2 x 16 x 16 positions by 1/127 of its block's maximum: 2e-3 of a gradient's largest entry is several of them."""
    from iprgan import _lib as L, engine as E
    from iprgan.ops import ConvSpec
    torch.manual_seed(3)
    c1, c2, bn, c3 = nn.Conv2d(3, 32, 3, 1, 1), nn.Conv2d(32, 32, 3, 1, 1), nn.BatchNorm2d(32), nn.Conv2d(32, 8, 3, 1, 1)
    with torch.no_grad():
        bn.weight.normal_(1, 0.2)
        bn.bias.normal_(0, 0.2)
    x, r = torch.randn(2, 3, 16, 16), torch.randn(2, 8, 16, 16)
    d = lambda t: t.detach().double()
    F = nn.functional
    a1 = F.leaky_relu(F.conv2d(d(x), d(c1.weight), d(c1.bias), padding=1), 0.2)
    a2 = F.conv2d(a1, d(c2.weight), d(c2.bias), padding=1)
    mean, var = a2.mean((0, 2, 3), keepdim=True), a2.var((0, 2, 3), unbiased=False, keepdim=True)
    inv = 1 / torch.sqrt(var + bn.eps)
    g, b = d(bn.weight).view(1, -1, 1, 1), d(bn.bias).view(1, -1, 1, 1)
    a3 = F.relu((a2 - mean) * inv * g + b)
    x8, a1q, a2q, a3q = (round8(t) for t in (d(x), a1, a2, a3))
    dy = d(r)
    want = {}
    want['c3'] = nn.grad.conv2d_weight(a3q, c3.weight.shape, dy, padding=1)
    g3 = nn.grad.conv2d_input(a3.shape, d(c3.weight), dy, padding=1)
    t = (a2q - mean) * inv
    dz = torch.where(t * g + b > 0, g3, torch.zeros_like(g3))
    want['bn'], want['bnb'] = (dz * t).sum((0, 2, 3)), dz.sum((0, 2, 3))
    M = 2 * 16 * 16
    g2 = g * inv * (dz - dz.sum((0, 2, 3), keepdim=True) / M - t * (dz * t).sum((0, 2, 3), keepdim=True) / M)
    want['c2'] = nn.grad.conv2d_weight(a1q, c2.weight.shape, g2, padding=1)
    g1 = nn.grad.conv2d_input(a1.shape, d(c2.weight), g2, padding=1) * torch.where(a1q > 0, 1.0, 0.2)
    want['c1'] = nn.grad.conv2d_weight(x8, c1.weight.shape, g1, padding=1)
    want['c1b'] = g1.sum((0, 2, 3))
    want['x'] = nn.grad.conv2d_input(x.shape, d(c1.weight), g1, padding=1)
    for m in (c1, c2, bn, c3):
        m.to(dev)
    plan = [E.ToNHWC(3), E.Conv(ConvSpec(3, 32, 3, 1, 1, act=L.ACT_LRELU, slope=0.2), c1), E.Conv(ConvSpec(32, 32, 3, 1, 1), c2),
            E.BatchNorm(bn, act=L.ACT_RELU), E.Conv(ConvSpec(32, 8, 3, 1, 1), c3), E.ToNCHW(8)]
    ckpt8(True)
    xin = x.to(dev).requires_grad_(True)
    (E.Chain(plan)(xin, True) * r.to(dev)).sum().backward()
    got = {'c3': c3.weight.grad, 'bn': bn.weight.grad, 'bnb': bn.bias.grad, 'c2': c2.weight.grad, 'c1': c1.weight.grad, 'c1b': c1.bias.grad,
           'x': xin.grad}
    for k, v in want.items():
        err = float((got[k].cpu().double() - v).abs().max() / v.abs().max())
        assert err <= 2e-3, (k, err)


NETS = ['ConvGenerator32', 'SNDiscriminator32', 'SRResNet', 'Discriminator96', 'Resnet6Blocks', 'ConvDiscriminator', 'VGG19Feature']
SHAPES = {'ConvGenerator32': (4, 128), 'SNDiscriminator32': (4, 3, 32, 32), 'SRResNet': (2, 3, 24, 24), 'Discriminator96': (2, 3, 96, 96),
          'Resnet6Blocks': (1, 3, 64, 64), 'ConvDiscriminator': (2, 3, 64, 64), 'VGG19Feature': (1, 3, 64, 64)}


@pytest.mark.parametrize('name', NETS)
@pytest.mark.parametrize('math', ['fp32', 'fp32x3', 'bf16act'], indirect=True)
def test_every_network_runs_with_checkpoints(dev, ckpt8, name, math):
    """Outputs are those of the plain pass, bit for bit; gradients point where the plain pass's point.

    How far they may turn: behind a ReLU of normal values a block of 32 has a maximum m of about 2.1 sigma and a step between m / 127.5
    and m / 63.75, on average m / 90.  A positive value below half a step - 0.0117 sigma, a share of 0.0117 * 0.4 = 0.47 % of all values,
    0.93 % of the positive ones - is stored as zero and loses its gradient.  n such masks in a row lose a share of 1 - (1 - 0.0093)^n of the
    gradient's energy and leave a cosine of the root of the rest; twice that share is granted.  (Masks of norm layers and of LeakyReLU lose
    less, the noise of the values themselves is 1e-5 of the energy.)"""
    if math == 'bf16act' and name not in ('ConvGenerator32', 'SNDiscriminator32'):
        pytest.skip('bf16act covers the DCGAN family')
    from iprgan import networks
    torch.manual_seed(5)
    net = getattr(networks, name)(**({'n_block': 2} if name == 'SRResNet' else {})).to(dev)
    net.train()
    state = {k: v.clone() for k, v in net.state_dict().items()}
    x = torch.randn(SHAPES[name], generator=torch.Generator().manual_seed(1)).to(dev)
    res = []
    for on in (False, True):
        net.load_state_dict(state)
        ckpt8(on)
        xin = x.clone().requires_grad_(True)
        for p in net.parameters():
            p.grad = None
        y = net(xin)
        r = torch.randn(y.shape, generator=torch.Generator().manual_seed(2)).to(dev)
        (y * r).sum().backward()
        res.append((y.detach().clone(), torch.cat([t.grad.flatten() for t in [xin, *net.parameters()] if t.grad is not None]).double()))
    assert torch.equal(res[0][0], res[1][0])
    a, b = res[0][1], res[1][1]
    assert bool(torch.isfinite(b).all())
    assert not torch.equal(a, b), 'the checkpoints were not used'
    cos = float((a * b).sum() / (a.norm() * b.norm()))
    masks = sum(1 for op in net.chain().ops for a in [getattr(op, 'act', op.out_act[0]), getattr(op, 'prelu', None)] if a)
    masks += sum(type(op).__name__ in ('PReLU', 'PixelShufflePReLU') for op in net.chain().ops)
    assert cos > (1 - 2 * (1 - (1 - 0.0093) ** max(masks, 1))) ** 0.5, (cos, masks)


def test_checkpoints_lower_the_peak_memory_of_a_pass(dev, ckpt8):
    from iprgan import engine, networks
    net = networks.SNDiscriminator64().to(dev)
    x = torch.randn(64, 3, 64, 64, device=dev)
    held = []
    for on in (False, True):
        ckpt8(on)
        torch.cuda.synchronize()
        base = torch.cuda.memory_allocated()
        y = net(x)
        held.append(torch.cuda.memory_allocated() - base)       # what the recorded pass keeps for its backward
        y.sum().backward()
        del y
    # fp32 activations to 1 + 1/32 bytes an element; the layers' small tensors stay
    assert held[1] < 0.35 * held[0], held


def test_graphed_step_with_checkpoints_is_bit_identical_to_eager(dev, ckpt8):
    from iprgan import Config, graphs, models
    ckpt8(True)
    runs = []
    for graphed in (False, True):
        torch.manual_seed(0)
        model = models.DCGAN(Config(cases.DCGAN_CFG), device=[dev])
        recipe.fill(model.G.module, 3)
        recipe.fill(model.D.module, 4)
        model.G.to(dev), model.D.to(dev)

        def body(s):
            model.update_d({'real_sample': s['x'], 'latent': s['z']})
            model.update_g({'fake_sample': model.fake_sample})
        first = {'x': torch.zeros(4, 3, 64, 64, device=dev), 'z': torch.zeros(4, 128, device=dev)}
        step = graphs.GraphedStep(model, body, first, warmup=2) if graphed else body
        for i in range(6):
            s = {'x': torch.tanh(recipe.tensor(7, 100 + i, (4, 3, 64, 64))).to(dev), 'z': recipe.tensor(7, 200 + i, (4, 128)).to(dev)}
            step(s)
            torch.cuda.synchronize()
        if graphed:
            assert step.graph is not None, step.failed
        runs.append([p.detach().clone() for p in list(model.G.parameters()) + list(model.D.parameters())])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.parametrize('math', ['fp32', 'fp32x3', 'bf16act'], indirect=True)
@pytest.mark.parametrize('batch', [1, 3, 70])
def test_generator_served_from_4_bit_dense_weights(dev, math, batch):
    """quantize_dense(): eval passes equal those of a generator whose Linear holds the rounded values; training passes keep fp32."""
    from iprgan import networks, ops
    torch.manual_seed(2)
    net, ref = networks.ConvGenerator32().to(dev), networks.ConvGenerator32().to(dev)
    ref.load_state_dict(net.state_dict())
    with torch.no_grad():
        w = ref.fc[0].weight
        w.copy_(ops.mx4_dequant(ops.mx4_quant(w)))
    z = torch.randn(batch, 128, generator=torch.Generator().manual_seed(1)).to(dev)
    assert net.quantize_dense() == 1
    net.eval(), ref.eval()
    for p in [*net.parameters(), *ref.parameters()]:
        p.requires_grad_(False)
    za, zb = z.clone().requires_grad_(True), z.clone().requires_grad_(True)
    a, b = net(za), ref(zb)
    tol = 2e-2 if math == 'bf16act' else 5e-4
    assert float((a - b).detach().abs().max()) <= tol * float(b.detach().abs().max())
    a.sum().backward(), b.sum().backward()
    # Two evaluations of the Linear differ by about 1e-6 of sigma.  Behind it a sample passes 8192 + 16384 + 32768 + 65536 = 123 k masks, and a
    # pre-activation lies within 1e-6 sigma of zero with probability 2e-6 * 0.4: 0.1 flipped masks a sample.  A flip turns one of those
    # terms of the sample's gradient on or off (1e-2, as everywhere in these tests); 70 samples have 7 expected flips, so a third of the rows
    # may hold one, the rest are 2e-3.
    err = (za.grad - zb.grad).abs().amax(1) / zb.grad.abs().max()
    one, flipped = (5e-2, 5e-2) if math == 'bf16act' else (2e-3, 1e-2)
    assert float(err.max()) <= flipped and int((err > one).sum()) <= (batch + 2) // 3, err
    net.train()
    plain = networks.ConvGenerator32().to(dev)
    plain.load_state_dict(net.state_dict())
    with torch.no_grad():
        assert torch.equal(net(z), plain(z))


def test_4_bit_dense_weights_refuse_what_they_cannot_do(dev):
    from iprgan import networks
    net = networks.ConvGenerator32().to(dev)
    z = torch.randn(2, 128, device=dev)
    net.quantize_dense()
    net.eval()
    with pytest.raises(RuntimeError, match='no weight gradient'):
        net(z).sum().backward()
    with torch.no_grad():
        net.fc[0].weight.mul_(2)
        with pytest.raises(RuntimeError, match='out of date'):
            net(z)
        net.quantize_dense()
        net(z)
        net.quantize_dense(False)
        net.fc[0].weight.mul_(2)
        net(z)
    with pytest.raises(RuntimeError, match='no dense layer'):
        networks.SRResNet(n_block=1).to(dev).quantize_dense()


def test_compression_attack(dev):
    from iprgan import Config, attacks, networks, ops, tools
    net = networks.ConvGenerator32()
    slm = tools.SignLossModel(net, Config({'gamma_0': 0.1, 'string': 'EXAMPLE A'}))
    net.to(dev), slm.to(dev)
    before = {k: v.detach().clone() for k, v in net.named_parameters()}
    nbytes, small = attacks.quantize_(net)
    assert nbytes == 4 * sum(v.numel() for v in before.values() if v.dim() >= 2) and small < nbytes / 4
    for k, p in net.named_parameters():
        if p.dim() < 2:
            assert torch.equal(p, before[k])
        else:
            w = before[k].cpu()
            r = R.mx4_decode(*R.mx4_encode(w.reshape(w.shape[0], -1)), w[0].numel())
            assert np.array_equal(p.detach().cpu().double().view(w.shape[0], -1).numpy(), r.numpy()), k
    assert float(slm.compute_ber(net)) == 0.0
    net(torch.randn(2, 128, device=dev))


def test_encoder_heads_served_from_4_bit_weights(dev):
    """Two dense layers behind the encoder's body; K = 2048 is one sum of 2048 terms: 2048 half steps of the terms' magnitude."""
    from iprgan import networks, ops
    torch.manual_seed(4)
    net, ref = networks.Encoder32().to(dev).eval(), networks.Encoder32().to(dev).eval()
    ref.load_state_dict(net.state_dict())
    assert net.quantize_dense() == 2
    with torch.no_grad():
        for m in (ref.q_mean, ref.q_logvar):
            m.weight.copy_(ops.mx4_dequant(ops.mx4_quant(m.weight)))
        x = torch.randn(5, 3, 32, 32, generator=torch.Generator().manual_seed(1)).to(dev)
        got, q = net(x)[1], ref.chain()[0](x, False).double()
        for a, m in zip(got, (ref.q_mean, ref.q_logvar)):
            w = m.weight.detach().double()
            want, mag = q @ w.t().contiguous() + m.bias.detach().double(), q.abs() @ w.abs().t().contiguous() + m.bias.detach().double().abs()
            assert bool(((a.double() - want).abs() <= 2048 * 2.0 ** -24 * mag).all())
    assert net.quantize_dense(False) == 2


def test_a_copied_or_moved_generator_is_served_as_before(dev):
    import copy
    from iprgan import networks
    torch.manual_seed(6)
    net = networks.ConvGenerator32().to(dev).eval()
    net.quantize_dense()
    z = torch.randn(3, 128, generator=torch.Generator().manual_seed(1)).to(dev)
    with torch.no_grad():
        want = net(z)
        twin = copy.deepcopy(net)
        assert torch.equal(twin(z), want)
        twin.fc[0].weight.mul_(2)
        with pytest.raises(RuntimeError, match='out of date'):
            twin(z)
        assert torch.equal(net.cpu().to(dev)(z), want)
        net.fc[0].weight.mul_(2)
        net.cpu().to(dev)
        with pytest.raises(RuntimeError, match='out of date'):
            net(z)


def test_a_small_channel_keeps_its_gradient(dev, ckpt8, monkeypatch):
    """conv + LeakyReLU -> conv, the channels of the first scaled over three decades, in blocks of 32: with `engine: {ckpt8: true}` the masks
    are those of the activations, so the first convolution's gradients, channel by channel, are those of the exact pass but for the
    rounding of its input: sum |g| |x - x8|, written out below, and 2^-14 of the magnitudes for the fp32 arithmetic, 288 + 512 roundings
    in a row at most, each half a step.  Of the second's gradients a channel's are off by at most a step of its blocks."""
    from iprgan import _lib as L, configs, engine as E
    from iprgan.ops import ConvSpec
    torch.manual_seed(9)
    c1, c2 = nn.Conv2d(4, 64, 3, 1, 1), nn.Conv2d(64, 32, 3, 1, 1)
    s = torch.logspace(0, -3, 64)[torch.randperm(64, generator=torch.Generator().manual_seed(1))]
    with torch.no_grad():
        c1.weight.mul_(s.view(-1, 1, 1, 1))
        c1.bias.mul_(s)
        c2.weight.div_(s.view(1, -1, 1, 1))                      # every channel matters to the second layer
    x, r = torch.randn(2, 4, 16, 16), torch.randn(2, 32, 16, 16)
    d = lambda t: t.detach().double()
    F = nn.functional
    a1 = F.leaky_relu(F.conv2d(d(x), d(c1.weight), d(c1.bias), padding=1), 0.2)
    dy = d(r)
    g1 = nn.grad.conv2d_input(a1.shape, d(c2.weight), dy, padding=1) * torch.where(a1 > 0, 1.0, 0.2)
    mag = nn.grad.conv2d_input(a1.shape, d(c2.weight).abs(), dy.abs(), padding=1)
    wantw, wantb = nn.grad.conv2d_weight(d(x), c1.weight.shape, g1, padding=1), g1.sum((0, 2, 3))
    x8 = round8(d(x))
    tolw = nn.grad.conv2d_weight((d(x) - x8).abs(), c1.weight.shape, g1.abs(), padding=1)
    tolw = tolw + 2.0 ** -14 * nn.grad.conv2d_weight(d(x).abs(), c1.weight.shape, mag, padding=1)
    tolb = 2.0 ** -14 * mag.sum((0, 2, 3))
    p = a1.permute(0, 2, 3, 1).reshape(-1, 32)
    _, sc = R.mx8_encode(p.float())
    step = torch.exp2(sc.double() - 127).repeat_interleave(32).view(2, 16, 16, 64).permute(0, 3, 1, 2)
    want2 = nn.grad.conv2d_weight(a1, c2.weight.shape, dy, padding=1)
    tol2 = nn.grad.conv2d_weight(step, c2.weight.shape, dy.abs(), padding=1) + 2.0 ** -14 * nn.grad.conv2d_weight(a1.abs(), c2.weight.shape, dy.abs(), padding=1)
    c1.to(dev), c2.to(dev)
    plan = [E.ToNHWC(4), E.Conv(ConvSpec(4, 64, 3, 1, 1, act=L.ACT_LRELU, slope=0.2), c1), E.Conv(ConvSpec(64, 32, 3, 1, 1), c2), E.ToNCHW(32)]
    for k in ('IPRGAN_CKPT8', 'IPRGAN_CKPT8_SIGNS'):             # (put back, with the module's switches, when the test ends)
        monkeypatch.setenv(k, '0')
    monkeypatch.delenv('IPRGAN_CKPT8_SIGNS')
    monkeypatch.setattr(E, '_CKPT8_SIGNS', False)
    ckpt8(False)
    configs.apply_engine({'engine': {'ckpt8': True}}, set_math=False)
    assert E._CKPT8 and E._CKPT8_SIGNS
    (E.Chain(plan)(x.to(dev), True) * r.to(dev)).sum().backward()
    for got, want, tol in ((c1.weight.grad, wantw, tolw), (c1.bias.grad, wantb, tolb), (c2.weight.grad, want2, tol2)):
        err = (got.cpu().double() - want).abs()
        assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize('name,math', [('SNDiscriminator32', 'fp32'), ('SNDiscriminator32', 'fp32x3'), ('SNDiscriminator32', 'bf16act'),
                                       ('VGG19Feature', 'fp32'), ('VGG19Feature', 'fp32x3')], indirect=['math'])
@pytest.mark.parametrize('least', [1, None])
def test_data_gradients_without_norm_layers_are_those_of_the_plain_pass(dev, ckpt8, monkeypatch, name, math, least):
    """Where every mask is read off an output and no layer's data gradient reads its input, a checkpoint with exact masks changes weight gradients
    only: the input's and the biases' are bit-identical, with every tensor packed and with the default threshold (some packed, some not).
    A weight gradient is off by the rounding of its layer's input: at most half a step of a block, m / 127.5 of its maximum m, a third of that on
    average, where the values' average is m / 4 and more: 2 % of a tensor's gradient if it is as incoherent as the rounding; 5 % granted."""
    from iprgan import engine, networks
    if least is None:
        monkeypatch.setattr(engine, '_CKPT8_MIN', 1 << 14)
    monkeypatch.setattr(engine, '_CKPT8_SIGNS', True)
    torch.manual_seed(5)
    net = getattr(networks, name)().to(dev)
    net.train()
    state = {k: v.clone() for k, v in net.state_dict().items()}
    x = torch.randn(SHAPES[name], generator=torch.Generator().manual_seed(1)).to(dev)
    res = []
    for on in (False, True):
        net.load_state_dict(state)
        ckpt8(on)
        xin = x.clone().requires_grad_(True)
        for p in net.parameters():
            p.grad = None
        y = net(xin)
        r = torch.randn(y.shape, generator=torch.Generator().manual_seed(2)).to(dev)
        (y * r).sum().backward()
        res.append({'x': xin.grad, **{k: p.grad for k, p in net.named_parameters() if p.grad is not None}})
    moved = 0
    for k, a in res[0].items():
        b = res[1][k]
        if k == 'x' or k.endswith('bias'):
            assert torch.equal(a, b), k
        else:
            moved += not torch.equal(a, b)
            assert float((a - b).norm()) <= 0.05 * float(a.norm()), k
    assert moved > 0 or len(res[0]) == 1, 'the checkpoints were not used'


def test_chain_of_packed_and_plain_tensors(dev, ckpt8, monkeypatch):
    """The default threshold in the middle of a chain: conv + LeakyReLU (16 384 elements: packed, masks kept) -> conv -> BatchNorm + ReLU (8 192: its
    input stays, its output is dropped all the same) -> conv, written out in float64.  Bounds as in the chain test above."""
    from iprgan import _lib as L, engine as E
    from iprgan.ops import ConvSpec
    torch.manual_seed(3)
    c1, c2, bn, c3 = nn.Conv2d(3, 32, 3, 1, 1), nn.Conv2d(32, 16, 3, 1, 1), nn.BatchNorm2d(16), nn.Conv2d(16, 8, 3, 1, 1)
    with torch.no_grad():
        bn.weight.normal_(1, 0.2)
        bn.bias.normal_(0, 0.2)
    x, r = torch.randn(2, 3, 16, 16), torch.randn(2, 8, 16, 16)
    d = lambda t: t.detach().double()
    F = nn.functional
    a1 = F.leaky_relu(F.conv2d(d(x), d(c1.weight), d(c1.bias), padding=1), 0.2)
    p = a1.permute(0, 2, 3, 1).contiguous()
    a1q = R.mx8_decode(*R.mx8_encode_signs(p.float())).view(p.shape).permute(0, 3, 1, 2).contiguous()
    a2 = F.conv2d(a1, d(c2.weight), d(c2.bias), padding=1)
    inv = 1 / torch.sqrt(a2.var((0, 2, 3), unbiased=False, keepdim=True) + bn.eps)
    t = (a2 - a2.mean((0, 2, 3), keepdim=True)) * inv
    g, b = d(bn.weight).view(1, -1, 1, 1), d(bn.bias).view(1, -1, 1, 1)
    a3 = F.relu(t * g + b)
    dy = d(r)
    want = {'c3': nn.grad.conv2d_weight(a3, c3.weight.shape, dy, padding=1)}
    dz = torch.where(t * g + b > 0, nn.grad.conv2d_input(a3.shape, d(c3.weight), dy, padding=1), 0.0)
    want['bn'], want['bnb'] = (dz * t).sum((0, 2, 3)), dz.sum((0, 2, 3))
    M = 2 * 16 * 16
    g2 = g * inv * (dz - dz.sum((0, 2, 3), keepdim=True) / M - t * (dz * t).sum((0, 2, 3), keepdim=True) / M)
    want['c2'] = nn.grad.conv2d_weight(a1q, c2.weight.shape, g2, padding=1)
    g1 = nn.grad.conv2d_input(a1.shape, d(c2.weight), g2, padding=1) * torch.where(a1 > 0, 1.0, 0.2)
    want['c1'], want['c1b'] = nn.grad.conv2d_weight(d(x), c1.weight.shape, g1, padding=1), g1.sum((0, 2, 3))
    want['x'] = nn.grad.conv2d_input(x.shape, d(c1.weight), g1, padding=1)
    for m in (c1, c2, bn, c3):
        m.to(dev)
    plan = [E.ToNHWC(3), E.Conv(ConvSpec(3, 32, 3, 1, 1, act=L.ACT_LRELU, slope=0.2), c1), E.Conv(ConvSpec(32, 16, 3, 1, 1), c2),
            E.BatchNorm(bn, act=L.ACT_RELU), E.Conv(ConvSpec(16, 8, 3, 1, 1), c3), E.ToNCHW(8)]
    ckpt8(True)
    monkeypatch.setattr(E, '_CKPT8_MIN', 1 << 14)
    monkeypatch.setattr(E, '_CKPT8_SIGNS', True)
    xin = x.to(dev).requires_grad_(True)
    (E.Chain(plan)(xin, True) * r.to(dev)).sum().backward()
    got = {'c3': c3.weight.grad, 'bn': bn.weight.grad, 'bnb': bn.bias.grad, 'c2': c2.weight.grad, 'c1': c1.weight.grad, 'c1b': c1.bias.grad,
           'x': xin.grad}
    for k, v in want.items():
        err = float((got[k].cpu().double() - v).abs().max() / v.abs().max())
        assert err <= 2e-3, (k, err)


@pytest.mark.parametrize('shuffle', [False, True])
def test_prelu_masks_are_those_of_the_plain_pass(dev, ckpt8, monkeypatch, shuffle):
    """conv -> (pixel shuffle) PReLU -> conv: the mask is read off the PReLU's input.  With exact masks the data gradient and the first convolution's
    gradients of it are bit-identical, the slope's is off by the rounding of x: sum |dy| step over the negative half at most."""
    from iprgan import engine as E
    from iprgan.ops import ConvSpec
    monkeypatch.setattr(E, '_CKPT8_SIGNS', True)
    torch.manual_seed(11)
    c1, pr, c2 = nn.Conv2d(4, 64, 3, 1, 1).to(dev), nn.PReLU().to(dev), nn.Conv2d(16 if shuffle else 64, 8, 3, 1, 1).to(dev)
    plan = [E.ToNHWC(4), E.Conv(ConvSpec(4, 64, 3, 1, 1), c1), E.PixelShufflePReLU(pr) if shuffle else E.PReLU(pr),
            E.Conv(ConvSpec(16 if shuffle else 64, 8, 3, 1, 1), c2), E.ToNCHW(8)]
    side = 32 if shuffle else 16
    x, r = torch.randn(2, 4, 16, 16).to(dev), torch.randn(2, 8, side, side).to(dev)
    res = []
    for on in (False, True):
        ckpt8(on)
        for m in (c1, pr, c2):
            m.zero_grad()
        xin = x.clone().requires_grad_(True)
        (E.Chain(plan)(xin, True) * r).sum().backward()
        res.append((xin.grad, c1.bias.grad, pr.weight.grad, c2.weight.grad))
    (xa, ba, sa, wa), (xb, bb, sb, wb) = res
    assert torch.equal(xa, xb) and torch.equal(ba, bb) and not torch.equal(wa, wb)
    with torch.no_grad():
        h = nn.functional.conv2d(x.double().cpu(), c1.weight.double().cpu(), c1.bias.double().cpu(), padding=1)
        g = nn.grad.conv2d_input((2, c2.in_channels, side, side), c2.weight.double().cpu(), r.double().cpu(), padding=1)
        bound = float(h.abs().max()) / 63.75 * float(g.abs().sum())
    assert abs(float(sa - sb)) <= bound


@pytest.mark.parametrize('name,math', [(n, m) for n in ('ConvGenerator32', 'SRResNet', 'Discriminator96', 'Resnet6Blocks', 'ConvDiscriminator')
                                       for m in ('fp32', 'fp32x3')] + [('ConvGenerator32', 'bf16act')], indirect=['math'])
def test_every_gradient_of_networks_with_norm_layers(dev, ckpt8, monkeypatch, name, math):
    """With exact masks a norm layer's data gradient depends on the rounding through its normalised input alone, and that through a sum that is small
    beside it; the parameters' gradients are sums over rounded factors as in the test above: each tensor by itself within the 5 % granted there.
    Left out: single numbers (a PReLU's slope: one sum, which may cancel) and biases below a norm layer (zero but for rounding)."""
    from iprgan import engine, networks
    monkeypatch.setattr(engine, '_CKPT8_SIGNS', True)
    torch.manual_seed(5)
    net = getattr(networks, name)(**({'n_block': 2} if name == 'SRResNet' else {})).to(dev)
    net.train()
    state = {k: v.clone() for k, v in net.state_dict().items()}
    x = torch.randn(SHAPES[name], generator=torch.Generator().manual_seed(1)).to(dev)
    res = []
    for on in (False, True):
        net.load_state_dict(state)
        ckpt8(on)
        xin = x.clone().requires_grad_(True)
        for p in net.parameters():
            p.grad = None
        y = net(xin)
        r = torch.randn(y.shape, generator=torch.Generator().manual_seed(2)).to(dev)
        (y * r).sum().backward()
        res.append({'x': xin.grad, **{k: p.grad for k, p in net.named_parameters()}})
    most = max(float(v.norm()) for v in res[0].values())
    for k, a in res[0].items():
        if a.numel() > 1 and float(a.norm()) > 1e-5 * most:
            err = float((a - res[1][k]).norm() / a.norm())
            assert err <= 0.05, (k, err)


def test_graphed_step_with_exact_masks_is_bit_identical_to_eager(dev, ckpt8, monkeypatch):
    from iprgan import engine
    monkeypatch.setattr(engine, '_CKPT8_SIGNS', True)
    test_graphed_step_with_checkpoints_is_bit_identical_to_eager(dev, ckpt8)
