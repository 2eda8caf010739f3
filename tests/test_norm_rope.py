"""norm_rope forward and backward against the formulas in 64 bits; refusals; replay from a captured graph."""
import math

import pytest
import torch

from deepof_amd.attention import rotary_frequencies
from sequence_common import DEVICES, DTYPES, TINY, U, U32, assert_within, draw, make_ops, strided


def reference(x, w, pos, freqs, eps, interleaved):
    """-> y and, for the bound, the size of the numbers each output is made of; 64 bits."""
    rot = 2 * len(freqs)
    r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) if w is not None else torch.ones_like(x[..., :1])
    y = x * r * (w if w is not None else 1.0)
    t = pos.double()[:, None, None] * freqs
    c, s = torch.cos(t), torch.sin(t)
    out, size = y.clone(), y.abs()
    a = slice(0, rot, 2) if interleaved else slice(0, rot // 2)
    b = slice(1, rot, 2) if interleaved else slice(rot // 2, rot)
    out[..., a] = y[..., a] * c - y[..., b] * s
    out[..., b] = y[..., b] * c + y[..., a] * s
    size[..., a] = size[..., b] = y[..., a].abs() + y[..., b].abs()
    return out, size


def reference_backward(g, x, w, pos, freqs, eps, interleaved):
    gy, _ = reference(g, None, -pos.double(), freqs, 0.0, interleaved)  # the inverse rotation turns the other way
    _, size = reference(g, None, -pos.double(), freqs, 0.0, interleaved)
    if w is None:
        return gy, size, None, None
    r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    xh = x * r
    dx = r * (w * gy - xh * (w * gy * xh).mean(-1, keepdim=True))
    dx_size = r * (w.abs() * size + xh.abs() * (w.abs() * size * xh.abs()).mean(-1, keepdim=True))
    return dx, dx_size, (gy * xh).sum((0, 1)), (size * xh.abs()).sum((0, 1))


# rows, query heads, key heads, head size, rotated part, interleaved, norm, memory order
CASES = [
    (1, 1, 1, 2, 2, False, True, "plain"),
    (1, 8, 2, 64, 64, False, True, "plain"),
    (5, 4, 4, 16, 16, False, True, "packed"),
    (7, 3, 1, 80, 40, True, True, "packed"),
    (13, 2, 2, 24, 12, False, True, "head_major"),
    (9, 6, 2, 128, 128, False, False, "plain"),
    (6, 5, 1, 96, 48, True, False, "odd"),
    (4, 2, 1, 128, 64, False, True, "odd"),
    (3, 2, 2, 200, 128, False, True, "odd"),      # two rounds of single elements per row
    (3, 2, 1, 256, 256, True, True, "plain"),
    (5, 2, 1, 6, 2, False, True, "plain"),
    (4, 2, 2, 32, 0, False, True, "plain"),       # norm without a rotation
    (300, 3, 1, 32, 32, False, True, "packed"),
]
EPS = 1e-5


def build(case, dtype, device, seed=0):
    n, hq, hk, d, rot, inter, norm, how = case
    g = torch.Generator().manual_seed(seed)
    t = dict(q=draw((n, hq, d), dtype, g, 1.5), k=draw((n, hk, d), dtype, g, 0.3), gq=draw((n, hq, d), dtype, g),
             gk=draw((n, hk, d), dtype, g))
    pos = torch.randint(-50, 2000000, (n,), generator=g, dtype=torch.int32)
    freqs = rotary_frequencies(rot, base=5e5) if rot else torch.zeros(0, dtype=torch.float64)
    w = [1.0 + 0.2 * torch.randn(d, generator=g) if norm else None for _ in range(2)]
    dev = {x: strided(v, device, how) for x, v in t.items()}
    kw = dict(q_weight=w[0].to(device) if norm else None, k_weight=w[1].to(device) if norm else None, eps=EPS, interleaved=inter)
    return t, pos, freqs, w, dev, kw


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("case", CASES, ids=str)
def test_forward_and_backward(device, dtype, case):
    n, hq, hk, d, rot, inter, norm, how = case
    ops = make_ops(device)
    t, pos, freqs, w, dev, kw = build(case, dtype, device)
    pd, fd = pos.to(device), freqs.to(device)
    got = dict(zip("qk", ops.norm_rope(dev["q"], dev["k"], pd, fd, **kw)))
    # fp32 in between: the sum of squares (a chain of at most 16 + 6 additions, halved by the root), root, division, two products,
    # the angle (half a turn in units of pi, 3 roundings) and the rotation's three operations stay below 32 roundings
    for i, x in enumerate("qk"):
        want, size = reference(t[x].double(), w[i].double() if norm else None, pos, freqs, EPS, inter)
        assert_within(x, got[x], want, U[dtype] * want.abs() * (1 + 2e-5) + 32 * U32 * size + TINY[dtype])
    back = ops.norm_rope_backward(dev["gq"], dev["gk"], dev["q"], dev["k"], pd, fd, **kw)
    for i, x in enumerate("qk"):
        dx, size, dw, dw_size = reference_backward(t["g" + x].double(), t[x].double(), w[i].double() if norm else None, pos, freqs,
                                                   EPS, inter)
        # as above, with the mean over the row (another 22) and its product
        assert_within("d" + x, back[i], dx, U[dtype] * dx.abs() * (1 + 2e-5) + 96 * U32 * size + TINY[dtype])
        if not norm:
            assert back[2 + i] is None
        else:  # a sum over n * heads terms, each good to 40 roundings: at most that many additions in a chain
            heads = (hq, hk)[i]
            assert_within("dw" + x, back[2 + i], dw, (n * heads + 40) * U32 * dw_size)


@pytest.mark.parametrize("device", DEVICES)
def test_gradient_against_differences(device):
    """d/dx of sum(y * g) by central differences of the 64-bit forward at a few elements, fp32 operator."""
    ops = make_ops(device)
    case = (4, 2, 1, 16, 8, False, True, "plain")
    t, pos, freqs, w, dev, kw = build(case, torch.float32, device, seed=3)
    dq = ops.norm_rope_backward(dev["gq"], dev["gk"], dev["q"], dev["k"], pos.to(device), freqs.to(device), **kw)[0].cpu().double()
    for e in ((0, 0, 0), (1, 1, 5), (3, 0, 15), (2, 1, 9)):
        vals = []
        for h in (1e-5, -1e-5):
            x = t["q"].double().clone()
            x[e] += h
            vals.append((reference(x, w[0].double(), pos, freqs, EPS, False)[0] * t["gq"].double()).sum())
        num = (vals[0] - vals[1]) / 2e-5  # truncation ~ h^2, cancellation ~ 2^-53 * 100 / 1e-5
        assert abs(float(num - dq[e])) < 2e-4 * max(1.0, abs(float(num)))


@pytest.mark.parametrize("device", DEVICES)
def test_in_place_and_no_rows(device):
    ops = make_ops(device)
    t, pos, freqs, w, dev, kw = build((9, 4, 2, 64, 64, False, True, "packed"), torch.bfloat16, device)
    pd, fd = pos.to(device), freqs.to(device)
    q, k = ops.norm_rope(dev["q"], dev["k"], pd, fd, **kw)
    q2, k2 = dev["q"].clone(), dev["k"].clone()
    ops.norm_rope(q2, k2, pd, fd, q_out=q2, k_out=k2, **kw)
    assert torch.equal(q, q2) and torch.equal(k, k2)
    none = ops.norm_rope(dev["q"][:0], dev["k"][:0], pd[:0], fd, **kw)
    assert none[0].shape == (0, 4, 64)
    back = ops.norm_rope_backward(dev["gq"][:0], dev["gk"][:0], dev["q"][:0], dev["k"][:0], pd[:0], fd, **kw)
    assert back[0].shape == (0, 4, 64) and float(back[2].abs().max()) == 0.0  # a sum over no rows


def test_frequencies():
    f = rotary_frequencies(8, base=10000.0)
    assert f.dtype == torch.float64 and torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-12)
    assert torch.allclose(rotary_frequencies(8, scale=4.0), f / 4.0, rtol=1e-15)
    part = rotary_frequencies(8, scale=4.0, original_length=2 * math.pi * 1000)  # turns 1000, 100, 10, 1
    want = f * torch.tensor([1.0, 1.0, (9 / 31) + (22 / 31) / 4, 0.25], dtype=torch.float64)
    assert torch.allclose(part, want, rtol=1e-12)
    for bad in (dict(rot_dim=3), dict(rot_dim=0), dict(rot_dim=4, scale=0.0), dict(rot_dim=4, base=-1.0),
                dict(rot_dim=4, scale=2.0, original_length=10.0, low_turns=5.0, high_turns=5.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(**bad)


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    from deepof_amd._capi import DofError
    ops = make_ops(device)
    t, pos, freqs, w, dev, kw = build((4, 2, 1, 16, 16, False, True, "plain"), torch.float32, device)
    q, k, pd, fd = dev["q"], dev["k"], pos.to(device), freqs.to(device)
    for args in ((q.double(), k, pd, fd), (q, k.half(), pd, fd), (q, k[:3], pd, fd), (q, k, pd.long(), fd), (q, k, pd, fd.float()),
                 (q, k, pd[:2], fd), (q[0], k, pd, fd), (q.transpose(1, 2), k, pd, fd), (q, k, pd, torch.zeros(9, dtype=torch.float64, device=device))):
        with pytest.raises(ValueError):
            ops.norm_rope(*args)
    with pytest.raises(ValueError):
        ops.norm_rope(q, k, pd, fd, q_weight=torch.ones(15, device=device))
    with pytest.raises(ValueError):
        ops.norm_rope(q, k, pd, fd, q_out=q[:1].expand(4, 2, 16))
    with pytest.raises(ValueError, match="share memory"):
        buf = torch.zeros(5, 2, 16, device=device)
        ops.norm_rope(buf[:4], k, pd, fd, q_out=buf[1:])
    with pytest.raises(ValueError):
        ops.norm_rope(q, k, pd, fd, eps=-1.0)
    with pytest.raises(DofError, match="head_dim"):
        z = torch.zeros(2, 1, 15, device=device)
        ops.norm_rope(z, z, pd[:2], fd[:2])
    with pytest.raises(DofError, match="head_dim"):
        z = torch.zeros(2, 1, 258, device=device)
        ops.norm_rope(z, z, pd[:2], fd[:2])


@pytest.mark.gpu
def test_weight_gradient_is_the_same_every_run_and_from_a_graph():
    ops = make_ops("cuda:0")
    t, pos, freqs, w, dev, kw = build((3001, 4, 2, 64, 64, False, True, "packed"), torch.bfloat16, "cuda:0")
    pd, fd = pos.cuda(), freqs.cuda()

    def step():
        q, k = ops.norm_rope(dev["q"], dev["k"], pd, fd, **kw)
        return (q, k) + ops.norm_rope_backward(dev["gq"], dev["gk"], dev["q"], dev["k"], pd, fd, **kw)

    eager = [x.clone() for x in step()]
    assert all(torch.equal(a, b) for a, b in zip(eager, step()))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        dev["q"].mul_(0.5 if i else 1.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))
