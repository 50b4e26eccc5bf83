"""CPU: refusals of the microscaled operators (their C entries check before they launch) and the checks of their containers."""
import ctypes as C

import pytest
import torch

import mx_forms
from iprgan import _lib as L
from iprgan import ops

P = C.c_void_p(4096)            # a non-null, aligned address: every call below is refused before anything is launched
ODD = C.c_void_p(4096 + 8)


def refused(name, *args):
    with pytest.raises(RuntimeError, match=name):
        L.call(name, *args)


def test_mx8_entries_refuse_bad_calls():
    refused('iprgan_mx8_quant', P, P, P, 0, 0, 0, None)
    refused('iprgan_mx8_quant', None, P, P, 8, 0, 0, None)
    refused('iprgan_mx8_quant', ODD, P, P, 8, 0, 0, None)
    refused('iprgan_mx8_quant', P, P, P, 8, 3, 0, None)
    refused('iprgan_mx8_quant', P, P, P, 8, 2, 4, None)
    refused('iprgan_mx8_dequant', P, P, P, 0, 0, 0, None)
    refused('iprgan_mx8_dequant', P, P, ODD, 8, 0, 0, None)
    refused('iprgan_mx8_dequant', P, P, P, 8, 2, 6, None)
    refused('iprgan_mx8_act_bwd', P, P, P, P, 8, 1, 0.0, 2, None)
    refused('iprgan_mx8_act_bwd', P, P, P, P, 0, 1, 0.0, 0, None)
    refused('iprgan_mx8_act_bwd', P, P, P, P, 8, 99, 0.0, 0, None)


def norm(codes=P, dy=P, gamma=P, beta=P, slope=None, dx=P, dgamma=P, dbeta=P, dslope=None, ws=P, G=1, M=8, C_=8, act=1, dbias=None, nb=0,
         kd=0, kx=0):
    return ('iprgan_mx8_norm_bwd', codes, P, dy, gamma, beta, P, P, slope, dx, dgamma, dbeta, dslope, ws, G, M, C_, act, 0.1, dbias, nb, 0.0,
            kd, 0, kx, 0, None)


@pytest.mark.parametrize('bad', [dict(M=0), dict(G=0), dict(C_=6), dict(codes=None), dict(ws=None), dict(dx=ODD), dict(act=3), dict(beta=None),
                                 dict(gamma=None, act=0), dict(dbeta=None), dict(dslope=P), dict(slope=P, act=1), dict(dslope=P, slope=P, act=2, G=2),
                                 dict(kd=1, kx=0), dict(kd=5, kx=5), dict(dbias=P, nb=9), dict(G=70000)])
def test_norm_backward_refuses(bad):
    refused(*norm(**bad))


def test_mx4_entries_refuse_bad_calls():
    assert L.query('iprgan_mx4_pitch', 1) == 4 and L.query('iprgan_mx4_pitch', 129) == 8 and L.query('iprgan_mx4_pitch', 0) == 0
    refused('iprgan_mx4_quant', P, P, P, 0, 4, 0, None)
    refused('iprgan_mx4_quant', P, P, P, 4, 0, 0, None)
    refused('iprgan_mx4_quant', P, ODD, P, 4, 4, 0, None)
    refused('iprgan_mx4_quant', P, P, P, 4, 4, 2, None)
    refused('iprgan_mx4_quant', P, P, P, 1 << 30, 1 << 10, 0, None)
    refused('iprgan_mx4_dequant', P, P, None, 4, 4, 0, None)
    lin = lambda *a: ('iprgan_mx4_linear',) + a
    refused(*lin(P, None, P, P, None, P, P, 0, 8, 8, 0, 0, 0.0, 0, None))
    refused(*lin(P, None, P, P, None, P, P, 8, 8, 0, 0, 0, 0.0, 0, None))
    refused(*lin(P, None, P, P, None, P, P, 8, 8, 8, 2, 0, 0.0, 0, None))            # a 4-bit x without scales
    refused(*lin(P, None, P, P, None, P, P, 8, 8, 8, 3, 0, 0.0, 0, None))
    refused(*lin(P, None, P, P, None, P, P, 8, 8, 8, 0, 9, 0.0, 0, None))
    refused(*lin(P, None, ODD, P, None, P, P, 8, 8, 8, 0, 0, 0.0, 0, None))
    refused(*lin(P, None, P, P, None, P, P, 8, 8, 8, 0, 0, 0.0, 2, None))
    refused(*lin(P, None, P, P, None, P, None, 4, 64, 8192, 0, 0, 0.0, 0, None))      # a split K needs its workspace
    refused('iprgan_mx4_linear_bwd', P, P, P, P, P, 8, 0, 8, 0, 0, None)
    refused('iprgan_mx4_linear_bwd', P, P, P, None, P, 8, 8, 8, 0, 0, None)
    refused('iprgan_mx4_linear_bwd', P, P, P, P, None, 4, 8192, 64, 0, 0, None)


def test_workspace_sizes():
    assert L.query('iprgan_mx4_linear_ws_floats', 0, 8, 8, 0, 0) == 0
    assert L.query('iprgan_mx4_linear_ws_floats', 4, 64, 8192, 0, 0) % (4 * 64) == 0
    assert L.query('iprgan_mx4_linear_ws_floats', 4, 64, 32, 0, 3) == 4 * 64 and L.query('iprgan_mx4_linear_ws_floats', 4, 64, 32, 0, 2) == 0
    assert L.query('iprgan_mx8_norm_bwd_ws_floats', 1, 100, 64) >= 5 * 64
    assert L.query('iprgan_mx8_norm_bwd_ws_floats', 0, 100, 64) == 0


def test_containers_refuse_what_does_not_fit():
    c8, s8 = torch.zeros(70, dtype=torch.int8), torch.zeros(3, dtype=torch.uint8)
    q = ops.Mx8(c8, s8, (2, 35))
    assert q.shape == (2, 35) and q.numel() == 70 and q.dim() == 2 and q.dtype == torch.float32
    assert q.view(7, 10).shape == (7, 10) and q.view((70,)).shape == (70,)
    for codes, scales, shape in ((c8, s8, (2, 36)), (c8, s8[:2], (70,)), (c8.int(), s8, (70,)), (c8, s8.int(), (70,))):
        with pytest.raises(RuntimeError, match='Mx8'):
            ops.Mx8(codes, scales, shape)
    with pytest.raises(RuntimeError, match='Mx8'):
        ops.Mx8(c8, s8, (70,), kind=3)
    c4, s4 = torch.zeros(3, 64, dtype=torch.uint8), torch.zeros(3, 4, dtype=torch.uint8)
    assert ops.Mx4(c4, s4, (3, 100)).shape == (3, 100)
    for codes, scales, shape in ((c4, s4, (3, 129)), (c4, s4, (2, 100)), (c4.int(), s4, (3, 100)), (c4, s4[:, :3], (3, 100))):
        with pytest.raises(RuntimeError, match='Mx4'):
            ops.Mx4(codes, scales, shape)


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 32)
    w4 = ops.Mx4(torch.zeros(3, 64, dtype=torch.uint8), torch.zeros(3, 4, dtype=torch.uint8), (3, 32))
    q = ops.Mx8(torch.zeros(128, dtype=torch.int8), torch.zeros(4, dtype=torch.uint8), (4, 32))
    for f in (lambda: ops.mx8_quant(x), lambda: ops.mx8_dequant(q), lambda: ops.mx4_quant(x), lambda: ops.mx4_dequant(w4),
              lambda: ops.mx4_linear(x, w4), lambda: ops.mx4_linear_bwd(torch.zeros(4, 3), w4), lambda: ops.act_bwd(x, q, 1),
              lambda: ops.bn_bwd(q, None, x, None, torch.zeros(32), torch.zeros(32), 0)):
        with pytest.raises(RuntimeError, match='GPU tensors'):
            f()


def test_shapes_are_checked():
    w4 = ops.Mx4(torch.zeros(3, 64, dtype=torch.uint8), torch.zeros(3, 4, dtype=torch.uint8), (3, 32))
    with pytest.raises(RuntimeError, match='mx4_linear'):
        ops.mx4_linear(torch.zeros(4, 33), w4)
    with pytest.raises(RuntimeError, match='mx4_linear'):
        ops.mx4_linear(torch.zeros(4, 32), torch.zeros(3, 32))
    with pytest.raises(RuntimeError, match='bias'):
        ops.mx4_linear(torch.zeros(4, 32), w4, torch.zeros(4))
    with pytest.raises(RuntimeError, match='mx4_linear_bwd'):
        ops.mx4_linear_bwd(torch.zeros(4, 32), w4)
    q = ops.Mx8(torch.zeros(128, dtype=torch.int8), torch.zeros(4, dtype=torch.uint8), (4, 32))
    with pytest.raises(RuntimeError, match='norm backward'):
        ops.bn_bwd(q, None, torch.zeros(4, 31), None, torch.zeros(32), torch.zeros(32), 0)
    with pytest.raises(RuntimeError, match='norm backward'):
        ops.bn_bwd(q, None, torch.zeros(4, 32), torch.zeros(31), torch.zeros(32), torch.zeros(32), 0)


def test_ckpt8_engine_key(monkeypatch):
    from iprgan import configs, engine
    monkeypatch.setenv('IPRGAN_CKPT8', '0')
    monkeypatch.setattr(engine, '_CKPT8', False)
    assert configs.apply_engine({'engine': {'ckpt8': True}}, set_math=False) == {'ckpt8': True} and engine._CKPT8
    configs.apply_engine({'engine': {'ckpt8': False}}, set_math=False)
    assert not engine._CKPT8


WRAP = 1 << 32          # added to a size: what an int would cut off


def refused_size(name, *args):
    """refused() by the entry's own checks: behind them there is no GPU here, and a launch fails too."""
    with pytest.raises(RuntimeError, match=name) as e:
        L.call(name, *args)
    assert 'launch failed' not in str(e.value), e.value


def test_sizes_past_an_int_are_not_cut():
    """A dimension of 2^32 + k is refused (or priced) as itself, never taken for k."""
    assert L.query('iprgan_mx4_pitch', WRAP + 128) == 0
    refused_size('iprgan_mx4_quant', P, P, P, 1, WRAP + 128, 0, None)
    refused_size('iprgan_mx4_quant', P, P, P, WRAP + 1, 128, 0, None)
    refused_size('iprgan_mx4_dequant', P, P, P, 1, WRAP + 128, 0, None)
    refused_size('iprgan_mx4_dequant', P, P, P, WRAP + 1, 128, 0, None)
    for i in range(3):
        d = [8, 8, 8]
        d[i] += WRAP
        refused_size('iprgan_mx4_linear', P, None, P, P, None, P, P, *d, 0, 0, 0.0, 0, None)
        refused_size('iprgan_mx4_linear_bwd', P, P, P, P, P, *d, 0, 0, None)
        assert L.query('iprgan_mx4_linear_ws_floats', *d, 0, 3) == 0 and L.query('iprgan_mx4_linear_bwd_ws_floats', *d, 0) == 0
    for bad in (dict(G=WRAP + 1), dict(M=WRAP + 8), dict(C_=WRAP + 8), dict(dbias=P, nb=WRAP + 8)):
        refused_size(*norm(**bad))
    assert L.query('iprgan_mx8_norm_bwd_ws_floats', 1, WRAP + 8, 8) == 0


def test_rows_of_a_map_are_within_the_limits():
    """All positions of a batch of maps are rows of one product: more than 2^20 are ordinary, 2^30 are refused, and so is a grid past a launch."""
    rows = 256 * 128 * 128
    assert L.query('iprgan_mx4_linear_ws_floats', rows, 4, 32, 0, 3) == rows * 4             # (tanh goes through the workspace)
    refused_size('iprgan_mx4_linear', P, None, P, P, None, P, P, 1 << 30, 8, 8, 0, 0, 0.0, 0, None)
    refused_size('iprgan_mx4_linear_bwd', P, P, P, P, P, 1 << 30, 8, 8, 0, 0, None)
    refused_size('iprgan_mx4_linear', P, None, P, P, None, P, P, 1 << 29, 1 << 20, 8, 0, 0, 0.0, 0, None)
    refused_size('iprgan_mx4_linear', P, None, P, P, None, P, P, 1 << 29, 255, 8, 0, 3, 0.0, 0, None)
    refused_size('iprgan_mx4_linear_bwd', P, P, P, P, P, 1 << 29, 8, 1 << 20, 0, 0, None)
    refused_size('iprgan_mx4_linear', P, P, P, P, None, P, P, 1 << 29, 1 << 23, 8, 2, 0, 0.0, 0, None)


@pytest.mark.parametrize('name,layers', [('ConvGenerator32', 1), ('ConvGenerator64', 1), ('Decoder32', 1), ('Encoder32', 2), ('SRResNet', 0)])
def test_quantize_dense_finds_the_dense_layers_of_every_network(name, layers):
    from iprgan import networks
    net = getattr(networks, name)()
    assert net.quantize_dense(False) == layers
    with pytest.raises(RuntimeError, match='GPU tensors' if layers else 'no dense layer'):
        net.quantize_dense()


def test_a_copied_or_moved_net_keeps_its_4_bit_copy():
    """The copy is keyed on the weights' storage and version: copying or moving a net changes the storage, not the weights.  A copy that was
    out of date stays so.  (Made by hand: quantising needs a GPU.)"""
    import copy
    import io
    from iprgan import networks
    net = networks.ConvGenerator32()
    op = net.chain().ops[0]

    def serve():
        n, k = op.weight.shape
        w4 = ops.Mx4(torch.randint(0, 256, (n, 64 * (k // 128)), dtype=torch.uint8), torch.full((n, k // 32), 120, dtype=torch.uint8), (n, k))
        op._mx4 = (op._weights_key(), w4, op.bias.detach().clone())
        return w4

    def pickled(n):
        f = io.BytesIO()
        torch.save(n, f)
        f.seek(0)
        return torch.load(f, weights_only=False)            # (a file this test has just written)

    w4 = serve()
    for twin in (copy.deepcopy(net), pickled(net)):
        t = twin.chain().ops[0]
        assert t.weight is not op.weight and t._mx4[0] == t._weights_key() != op._mx4[0]
        assert torch.equal(t._mx4[1].codes, w4.codes) and t._mx4[1].codes.data_ptr() != w4.codes.data_ptr() and t._mx4[1].shape == w4.shape
    with torch.no_grad():
        twin.fc[0].weight.mul_(2)
    assert t._mx4[0] != t._weights_key()
    again = copy.deepcopy(twin).chain().ops[0]
    assert again._mx4[0] != again._weights_key(), 'an outdated copy must not become valid'
    net._apply(lambda p: p.clone())                          # what .to() / .cuda() do
    assert op._mx4[0] == op._weights_key() and torch.equal(op._mx4[1].codes, w4.codes)
    with torch.no_grad():
        net.fc[0].weight.mul_(2)
    net._apply(lambda p: p.clone())
    assert op._mx4[0] != op._weights_key(), 'an outdated copy must not become valid'
    assert op._weights_key() == op._weights_key()
    serve()
    net.double()
    assert op._mx4[0] != op._weights_key(), 'another type: other weights'


def test_containers_are_rebuilt_through_their_checks():
    import copy
    q = ops.Mx8(torch.arange(64, dtype=torch.int8), torch.full((2,), 120, dtype=torch.uint8), (4, 16), ops.ST_BF16)
    t = copy.deepcopy(q)
    assert torch.equal(t.codes, q.codes) and torch.equal(t.scales, q.scales) and (t.shape, t.kind, t.get_device()) == ((4, 16), ops.ST_BF16, -1)


def test_ckpt8_signs_go_with_ckpt8_unless_set(monkeypatch):
    import os
    from iprgan import configs, engine
    monkeypatch.setenv('IPRGAN_CKPT8', '0')
    monkeypatch.delenv('IPRGAN_CKPT8_SIGNS', raising=False)
    monkeypatch.setattr(engine, '_CKPT8', False)
    monkeypatch.setattr(engine, '_CKPT8_SIGNS', False)
    for blk, want in (({'ckpt8': True}, True), ({'ckpt8': False}, False), ({'graph': False}, False)):
        configs.apply_engine({'engine': blk}, set_math=False)
        assert engine._CKPT8_SIGNS == want and 'IPRGAN_CKPT8_SIGNS' not in os.environ
    monkeypatch.setenv('IPRGAN_CKPT8_SIGNS', '0')
    configs.apply_engine({'engine': {'ckpt8': True}}, set_math=False)
    assert engine._CKPT8 and not engine._CKPT8_SIGNS
    configs.apply_engine({'engine': {'ckpt8': True, 'ckpt8_signs': True}}, set_math=False)
    assert engine._CKPT8_SIGNS


def test_mx8_quant_takes_the_signs_flag_beside_a_storage_kind():
    refused_size('iprgan_mx8_quant', P, P, P, 8, 16 | 3, 0, None)
    refused_size('iprgan_mx8_quant', P, P, P, 8, 32, 0, None)
    refused_size('iprgan_mx8_dequant', P, P, P, 8, 16, 0, None)


@pytest.mark.parametrize('gradient', [0, 1])
def test_sizes_of_the_form_tests_take_their_forms(gradient):
    kinds = {'f32': 0, 'bf16': 1, 'mx4': 2}
    form = (C.c_int * 5)()
    for kind, (M, K, N), want in mx_forms.GRADIENT if gradient else mx_forms.PRODUCT:
        L.call('iprgan_mx4_form', M, N, K, kinds[kind], gradient, form)
        assert tuple(form[:4]) + (form[4] > 1,) == want, (kind, M, K, N, tuple(form))
    refused_size('iprgan_mx4_form', 8, 8, 0, 0, gradient, form)
    refused_size('iprgan_mx4_form', 8, 8, 8, 3 - gradient, gradient, form)
    refused_size('iprgan_mx4_form', 8, 8, 8, 0, gradient, None)


def test_a_plain_bf16_tensor_is_not_taken_for_three_planes():
    """In 'fp32x3' mode a bf16 tensor is the first of three planes in one storage; one whose storage ends behind its own elements is refused before
    anything reads on."""
    before = L.get_math()
    L.set_math('fp32x3')
    try:
        x = torch.zeros(6, 32, dtype=torch.bfloat16)
        w4 = ops.Mx4(torch.zeros(32, 64, dtype=torch.uint8), torch.zeros(32, 4, dtype=torch.uint8), (32, 32))
        q = ops.Mx8(torch.zeros(192, dtype=torch.int8), torch.zeros(6, dtype=torch.uint8), (6, 32))
        v = torch.zeros(32)
        calls = (lambda t: ops.mx8_quant(t), lambda t: ops.mx4_quant(t), lambda t: ops.mx4_linear(t, w4), lambda t: ops.mx4_linear_bwd(t, w4),
                 lambda t: ops.act_bwd(t, q, 1), lambda t: ops.bn_bwd(q, None, t, v, v, v, 1, beta=v))
        whole = torch.zeros(3, 6, 32, dtype=torch.bfloat16)[0]
        slice_ = torch.zeros(3, 9, 32, dtype=torch.bfloat16)[0][3:]
        for f in calls:
            with pytest.raises(RuntimeError, match='three planes'):
                f(x)
            for t in (whole, slice_):
                with pytest.raises(RuntimeError, match='GPU tensors'):
                    f(t)
    finally:
        L.set_math(before)


def test_mx8_quant_norm_refuses_bad_calls():
    args = dict(x=P, codes=P, scales=P, gamma=P, beta=P, mean=P, invstd=P, ws=P, G=1, M=8, C=8, kind=0, ps=0)
    for bad in (dict(x=None), dict(ws=None), dict(mean=None), dict(gamma=None), dict(beta=None), dict(x=ODD), dict(codes=ODD), dict(ws=ODD), dict(M=0), dict(C=6),
                dict(kind=3), dict(kind=16), dict(kind=2, ps=8), dict(G=70000), dict(M=WRAP + 8), dict(C=WRAP + 8), dict(G=WRAP + 1)):
        refused_size('iprgan_mx8_quant_norm', *{**args, **bad}.values(), None)
