"""Plain CPU forms of the microscaled formats (csrc/mx8.hip, csrc/mx4.hip) in float64: what the tests compare against."""
import torch

LEVELS = torch.tensor([0., .5, 1., 1.5, 2., 3., 4., 6.], dtype=torch.float64)


def exponents(amax, half_open, cap):
    """Smallest e in [-127, cap] with amax < half_open * 2^e (half_open: where rounding would pass the largest code)."""
    e = torch.full(amax.shape, -127, dtype=torch.int64)
    for v in range(-127, cap):                                   # counting up, not a logarithm: exact and independent
        e += (amax >= half_open * 2.0 ** v).long() * (e == v).long()
    return e


def mx8_encode(x):
    """float32 / bfloat16 tensor -> (codes int8 [n], scales uint8 [ceil(n / 32)])"""
    v = x.detach().cpu().double().reshape(-1)
    n = v.numel()
    p = torch.zeros(-(-n // 32) * 32, dtype=torch.float64)
    p[:n] = v
    p = p.view(-1, 32)
    bad = ~torch.isfinite(p).all(1)
    p = torch.where(bad[:, None], torch.zeros_like(p), p)
    e = exponents(p.abs().amax(1), 127.5, 121)
    q = torch.round(p * torch.exp2(-e.double())[:, None]).clamp(-127, 127)        # torch.round: ties to even
    s = torch.where(bad, torch.full_like(e, 255), e + 127)
    return q.view(-1)[:n].to(torch.int8), s.to(torch.uint8)


def mx8_decode(codes, scales):
    """-> float64 [n]"""
    n = codes.numel()
    step = torch.exp2(scales.double() - 127)
    step[scales == 255] = float('nan')
    return codes.double() * step.repeat_interleave(32)[:n]


def mx4_encode(x):
    """[R, C] -> (codes uint8 [R, KB * 16], scales uint8 [R, KB])"""
    x = x.detach().cpu().double()
    r, c = x.shape
    p = torch.zeros(r, -(-c // 128) * 128, dtype=torch.float64)
    p[:, :c] = x
    p = p.view(r, -1, 32)
    bad = ~torch.isfinite(p).all(2)
    p = torch.where(bad[..., None], torch.zeros_like(p), p)
    e = exponents(p.abs().amax(2), 7.0, 125)
    y = p * torch.exp2(-e.double())[..., None]
    a = y.abs()
    idx = torch.zeros(a.shape, dtype=torch.int64)
    for i in range(1, 8):
        mid = (LEVELS[i - 1] + LEVELS[i]) / 2
        idx += (a >= mid).long() if i % 2 == 0 else (a > mid).long()       # a tie goes to the even code
    nib = (idx | (torch.signbit(y).long() << 3)).view(r, -1, 2)
    s = torch.where(bad, torch.full_like(e, 255), e + 127)
    return (nib[..., 0] | (nib[..., 1] << 4)).to(torch.uint8), s.to(torch.uint8)


def mx4_decode(codes, scales, cols):
    """-> float64 [R, cols]"""
    lut = torch.cat([LEVELS, -LEVELS])
    c = codes.cpu().long()
    v = torch.stack([lut[c & 15], lut[c >> 4]], 2).view(c.shape[0], -1, 32)
    step = torch.exp2(scales.cpu().double() - 127)
    step[scales.cpu() == 255] = float('nan')
    return (v * step[..., None]).reshape(c.shape[0], -1)[:, :cols]


def act(v, kind, slope):
    if kind == 1:
        return torch.where(v > 0, v, torch.zeros_like(v))
    if kind == 2:
        return torch.where(v > 0, v, v * slope)
    if kind == 3:
        return torch.tanh(v)
    if kind == 4:
        return torch.sigmoid(v) * 2 - 1
    return v


def mx8_encode_signs(x):
    """mx8_encode with no positive element rounded to zero (a block that holds a NaN or an infinity: all zero codes, as there)."""
    codes, s = mx8_encode(x)
    v = x.detach().cpu().double().reshape(-1)
    lost = (v > 0) & (codes == 0) & (s.repeat_interleave(32)[:v.numel()] != 255)
    return torch.where(lost, torch.ones_like(codes), codes), s


def mx8_encode_norm(x, gamma, beta, mean, invstd):
    """mx8_encode of a norm layer's input [G, M, C] with no element carried across v = 0, v = gamma (x - mean) invstd + beta: such an element goes one
    code further on its own side.  -> codes, scales, v > 0"""
    codes, s = mx8_encode(x)
    G, M, C = x.shape
    step = torch.exp2(s.double() - 127).repeat_interleave(32)[:codes.numel()].view(x.shape)
    k = (gamma.double() if gamma is not None else torch.ones(C, dtype=torch.float64)).view(1, 1, C) * invstd.double().view(G, 1, C)
    b = (beta.double() if beta is not None else torch.zeros(C, dtype=torch.float64)).view(1, 1, C)
    v = lambda t: (t - mean.double().view(G, 1, C)) * k + b
    q = codes.double().view(x.shape)
    want, got = v(x.double()) > 0, v(q * step) > 0
    up = torch.where(k < 0, -1.0, 1.0).expand(x.shape)
    q = torch.where(want & ~got, q + up, torch.where(got & ~want, q - up, q)).clamp(-127, 127)
    q = torch.where((s == 255).repeat_interleave(32)[:codes.numel()].view(x.shape), 0.0, q)
    return q.to(torch.int8).reshape(-1), s, want
