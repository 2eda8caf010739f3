"""Edges of the sequence operators: long tails of a softmax, long sums, what a row must not see, memory they may not touch, limits.
Every bound is derived where it stands; u is half a step of the type, relative to the value."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from deepof_amd import _capi
from sequence_common import DEVICES, DTYPES, TINY, U, U32, make_ops


def sink(n, gap, dtype):
    """One query of n keys: the first scores ``gap`` above the others.  Values 0 there, 1 elsewhere; what the output is to be."""
    q, k, v = torch.zeros(1, 1, 16), torch.zeros(n, 1, 16), torch.ones(n, 1, 16)
    q[0, 0, 0], k[0, 0, 0], v[0] = 1.0, 4.0 * gap, 0.0  # scale 1 / 4
    q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
    p = torch.softmax(k[:, 0, 0].double() / 4.0, 0)
    return q, k, v, float(p[1:].sum()), float(torch.logsumexp(k[:, 0, 0].double() / 4.0, 0))


# n weights that are each rounded by half a step of the type (fp16: or by 2^-36 of the largest, which is the sink's, nearly 1) and
# carry an exponent good to 32 fp32 roundings; a product takes 16 keys at a time, so their sum is a chain of n / 16 additions
def sink_bound(want, n, dtype):
    small = n * 2.0 ** -36 if dtype == torch.float16 else 0.0
    return want * (U[dtype] + (1 + U[dtype]) * (U[dtype] + (64 + n / 16) * U32)) + small + TINY[dtype]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES[1:], ids=str)
@pytest.mark.parametrize("n,gap", [(4096, 15.5), (8192, 17.5), (1500, 11.0)])
def test_long_tail_behind_a_sink(device, dtype, n, gap):
    ops = make_ops(device)
    q, k, v, want, lse = sink(n, gap, dtype)
    o, l = ops.attention(ops.attention_plan([1], [n]), q.to(device), k.to(device), v.to(device))
    assert float((o.cpu().double() - want).abs().max()) <= sink_bound(want, n, dtype)
    assert abs(float(l) - lse) <= 64 * U32 * lse


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES[1:], ids=str)
def test_very_long_tail_behind_a_sink(dtype):
    ops = make_ops("cuda:0")
    q, k, v, want, lse = sink(65536, 17.4, dtype)
    o, _ = ops.attention(ops.attention_plan([1], [65536]), q.cuda(), k.cuda(), v.cuda())
    assert float((o.cpu().double() - want).abs().max()) <= sink_bound(want, 65536, dtype)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES[1:], ids=str)
@pytest.mark.parametrize("n,gap", [(1000, 16.5), (3000, 17.0)])  # one part, and several
def test_step_with_a_long_tail_behind_a_sink(device, dtype, n, gap):
    ops = make_ops(device)
    q, k, v, want, _ = sink(n, gap, dtype)
    pages = -(-n // 100)
    kc, vc = (torch.zeros(pages * 100, 1, 16, dtype=dtype) for _ in range(2))
    kc[:n - 1], vc[:n - 1] = k[:-1], v[:-1]
    kc, vc = (x.view(pages, 100, 1, 16).to(device) for x in (kc, vc))
    table = torch.arange(pages, dtype=torch.int32, device=device)[None]
    o = ops.attention_step(q[None].to(device), k[None, -1:].to(device), v[None, -1:].to(device), kc, vc, table,
                           torch.tensor([n - 1], dtype=torch.int32, device=device))
    assert float((o.cpu().double() - want).abs().max()) <= sink_bound(want, n, dtype)


def plan_at(ops, q_off, k_off, causal, device):
    """A plan through the C ABI, whose documents may begin behind row 0 -> the record and its table on the device."""
    q_off, k_off = np.asarray(q_off, dtype=np.int64), np.asarray(k_off, dtype=np.int64)
    plan = _capi.AttnPlan()
    _capi.check(ops.lib, ops.lib.dof_attn_plan_size(len(q_off) - 1, q_off.ctypes.data, k_off.ctypes.data, causal, C.byref(plan)), "size")
    host = torch.empty(max(16, plan.table_bytes), dtype=torch.uint8)
    _capi.check(ops.lib, ops.lib.dof_attn_plan_table(C.byref(plan), q_off.ctypes.data, k_off.ctypes.data, 0, host.data_ptr()), "table")
    return plan, host.to(device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("lens", [[40], [200, 33], [20]])  # flat key tiles, tall ones, a document of the small kernel's
def test_rows_before_the_first_document_stay(device, dtype, lens):
    """First offsets above 0: the rows before are neither read (NaN) nor written, the gradients are those of the batch alone."""
    ops = make_ops(device)
    lead, hq, hk, d = 8, 4, 1, 16
    n = lead + sum(lens)
    g = torch.Generator().manual_seed(2)
    t = {x: torch.randn(n, h, d, generator=g).to(dtype).to(device) for x, h in (("q", hq), ("k", hk), ("v", hk), ("g", hq))}
    alone = {x: y[lead:].contiguous() for x, y in t.items()}
    whole = ops.attention_plan(lens, causal=True)
    o, lse = ops.attention(whole, alone["q"], alone["k"], alone["v"])
    want = dict(zip(("dq", "dk", "dv"), ops.attention_backward(whole, alone["g"], alone["q"], alone["k"], alone["v"], o, lse)), o=o, lse=lse)
    for x in t.values():
        x[:lead] = float("nan")
    off = lead + np.concatenate(([0], np.cumsum(lens)))
    plan, table = plan_at(ops, off, off, 1, device)
    out = {x: torch.full((n, h, d), 7.0, dtype=dtype, device=device) for x, h in (("o", hq), ("dq", hq), ("dk", hk), ("dv", hk))}
    out["lse"] = torch.full((n, hq), 7.0, device=device)
    st = {x: (h * d, d) for x, h in (("q", hq), ("k", hk))}
    rec = _capi.PACK_ATTENTION.pack(_capi.DTYPE_F32 + DTYPES.index(dtype), d, hq, hk, d ** -0.5, 0.0, *st["q"], *st["k"], *st["k"], *st["q"],
                                    *st["q"], *st["q"], *st["k"], *st["k"])
    p = {x: y.data_ptr() for x, y in (*t.items(), *out.items())}
    ops._launch("dof_attention_forward", C.byref(plan), table.data_ptr(), rec, p["q"], p["k"], p["v"], 0, p["o"], p["lse"])
    need = ops._bytes("dof_attention_workspace_bytes", C.byref(plan), rec)
    ws = torch.full((max(16, need) // 4,), 123.0, device=device)
    ops._launch("dof_attention_backward", C.byref(plan), table.data_ptr(), rec, p["g"], p["q"], p["k"], p["v"], 0, p["o"], p["lse"], p["dq"],
                p["dk"], p["dv"], ws.data_ptr())
    for x, y in out.items():
        assert bool((y[:lead] == 7).all()), x
        assert torch.equal(y[lead:], want[x]), x


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("hq,hk", [(2, 2), (4, 1)])  # a key head's query heads in one workgroup, and shared out
@pytest.mark.parametrize("keys", [[50], [3], [0, 200]])
def test_keys_without_any_query_row(device, hq, hk, keys):
    ops = make_ops(device)
    q, k, v = (torch.randn(n, h, 16).to(device) for n, h in ((0, hq), (sum(keys), hk), (sum(keys), hk)))
    plan = ops.attention_plan([0] * len(keys), keys)
    o, lse = ops.attention(plan, q, k, v)
    dq, dk, dv = ops.attention_backward(plan, q, q, k, v, o, lse)
    assert o.shape == dq.shape == (0, hq, 16) and lse.shape == (0, hq)
    assert dk.shape == dv.shape == k.shape and bool((dk == 0).all()) and bool((dv == 0).all())


@pytest.mark.gpu
def test_a_dropped_plan_stays_until_the_streams_that_use_it_are_done():
    """Made on the default stream, used on another one that is still busy: the block of its tiles is not handed out again before."""
    ops = make_ops("cuda:0")
    q, k, v = (torch.randn(75, 2, 32, device="cuda:0") for _ in range(3))
    plan = ops.attention_plan([40, 35], causal=True)
    want = [x.clone() for x in ops.attention(plan, q, k, v)]
    big = torch.randn(8192, 8192, device="cuda:0")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(20):
            big = big @ big * 1e-4
        got = ops.attention(plan, q, k, v)
    at, size = plan.table.data_ptr(), plan.table.numel()
    del plan
    others = [torch.empty(size, dtype=torch.uint8, device="cuda:0") for _ in range(64)]
    assert side.query() or all(x.data_ptr() != at for x in others)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("cap", [0.0, 4.0])
def test_a_row_depends_on_what_it_sees_alone(device, dtype, cap):
    """To the last bit: a later frame's key and value, made large and not, reach no earlier row, and a row's query no other row --
    forward, backward and step."""
    ops = make_ops(device)
    g = torch.Generator().manual_seed(4)
    n, d = 62, 16
    t = [(torch.randn(n, 2, d, generator=g) * 0.5).to(dtype).to(device) for _ in range(4)]
    plan = ops.attention_plan([n], causal=True)

    def run(q, k, v, do):
        o, lse = ops.attention(plan, q, k, v, cap=cap)
        return (o, lse) + ops.attention_backward(plan, do, q, k, v, o, lse, cap=cap)

    want = run(*t)
    last = n - 1
    for which, factor in ((0, 60.0), (1, 60.0), (2, 30.0), (0, 9.0), (1, 9.0)):
        x = [y.clone() for y in t]
        x[which][last] *= factor
        got = run(*x)
        assert torch.equal(got[0][:last], want[0][:last]) and torch.equal(got[1][:last], want[1][:last])
        assert torch.equal(got[2][:last], want[2][:last])  # dq

    def step(q, k, v):
        kc, vc = (torch.zeros(5, 16, 2, d, dtype=dtype, device=device) for _ in range(2))
        kc.view(80, 2, d)[:50], vc.view(80, 2, d)[:50] = t[1][:50], t[2][:50]
        return ops.attention_step(q, k, v, kc, vc, torch.arange(5, dtype=torch.int32, device=device)[None],
                                  torch.tensor([50], dtype=torch.int32, device=device), cap=cap)

    new = [x[None, 50:] for x in t[:3]]
    want = step(*new)
    for which in (0, 1, 2):
        x = [y.clone() for y in new]
        x[which][:, -1] *= 60.0
        assert torch.equal(step(*x)[:, :-1], want[:, :-1])


def test_cap_polynomial():
    """The odd polynomial that stands for tanh below 0.6, with its coefficients as stored: relative error below 1.5e-8."""
    x = np.linspace(1e-6, 0.6, 200001)
    y = x * x
    c = [float(np.float32(f)) for f in (-0.006276387721300125, 0.021116213873028755, -0.053875137120485306, 0.13332924246788025,
                                        -0.3333333134651184)]
    p = x * (1.0 + y * (c[4] + y * (c[3] + y * (c[2] + y * (c[1] + y * c[0])))))
    assert np.abs(p / np.tanh(x) - 1.0).max() < 1.5e-8


def equal_terms(n, d=8, heads=1):
    """Equal weights and values whose products and sums fp32 cannot hold: every rounding has the same sign over long stretches."""
    gen = torch.Generator().manual_seed(12)
    return 0.1 + 0.01 * torch.rand(1, heads, d, generator=gen).expand(n, heads, d)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n,d,few", [(4096, 8, 1), (16384, 16, 1), (3001, 72, 1), (1500, 40, 130)])
def test_long_float32_sums_of_one_sign(device, n, d, few):
    """o, dq and the sum behind it over n keys; dk and dv over n rows; few: rows (keys) on the other side, flat tiles or tall ones."""
    ops = make_ops(device)
    # a chain of at most 128 additions (256 where they take one term each, as in the emulation), n / 256 of those in a second one, and
    # 64 for weights, scores and the division, all of one sign
    rel = (256 + n / 256 + 64) * U32
    q, k, v = torch.zeros(few, 1, d), torch.zeros(n, 1, d), equal_terms(n, d).contiguous()
    plan = ops.attention_plan([few], [n])
    o, lse = ops.attention(plan, q.to(device), k.to(device), v.to(device))
    assert float((o.cpu().double() / v[:1].double() - 1).abs().max()) <= rel
    assert float((lse.cpu().double() - math.log(n)).abs().max()) <= 4 * U32 * math.log(n)
    # keys whose first half carries values 1 + v and the second v: dP differs by one between the halves, dS = +- 1 / (4 n) as the
    # weights are equal; k = +- (0.1 ..) makes every term of dq positive
    v2 = torch.zeros_like(v)
    half = n // 2
    v2[:half, :, 0] = 1.0
    kk = equal_terms(n, d).contiguous()
    kk[half:] *= -1.0
    g = torch.zeros(few, 1, d)
    g[..., 0] = 1.0
    f = half / n  # dS of the first half: (1 - f) / n, of the second: - f / n
    o2, lse2 = ops.attention(plan, q.to(device), kk.to(device), v2.to(device))
    dq = ops.attention_backward(plan, g.to(device), q.to(device), kk.to(device), v2.to(device), o2, lse2)[0]
    want = (f * (1 - f) + (1 - f) * f) * kk[:1].double() * d ** -0.5
    # dS itself: 1 - delta, delta good to rel, so relative 2 rel; the weights to 64 roundings
    assert float((dq.cpu().double() / want - 1).abs().max()) <= 4 * rel
    # n rows over 2 few keys: dv = sum of g / (2 few), dk = sum of dS q scale with dS = +- g . (v0 - v1) / (4 few)
    q3, g3 = equal_terms(n, d).contiguous(), equal_terms(n, d).contiguous()
    k3, v3 = torch.zeros(2 * few, 1, d), torch.zeros(2 * few, 1, d)
    v3[:few, 0, 0] = 1.0
    plan = ops.attention_plan([n], [2 * few])
    args = [x.to(device) for x in (q3, k3, v3)]
    o3, lse3 = ops.attention(plan, *args)
    dq3, dk3, dv3 = ops.attention_backward(plan, g3.to(device), *args, o3, lse3)
    want = g3[:1].double() * n / (2 * few)
    assert float((dv3.cpu().double() / want - 1).abs().max()) <= rel
    want = g3[0, 0, 0].double() / (4 * few) * n * q3[:1].double() * d ** -0.5
    for at, sign in ((slice(0, few), 1), (slice(few, None), -1)):
        assert float((dk3[at].cpu().double() * sign / want - 1).abs().max()) <= 4 * rel


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("d,new", [(8, 1), (72, 1), (40, 12), (128, 16)])
def test_step_whose_table_is_far_longer_than_its_streams(device, d, new):
    """The kernels for long sums, at lengths that need none of it."""
    ops = make_ops(device)
    g = torch.Generator().manual_seed(13)
    q, k, v = (torch.randn(2, new, 2, d, generator=g).to(device) for _ in range(3))
    kc, vc = (torch.randn(4, 256, 2, d, generator=g).to(device) for _ in range(2))
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32)
    lengths = torch.tensor([300, 470], dtype=torch.int32, device=device)
    outs = []
    for columns in (2, 1 << 17):
        t = torch.full((2, columns), -1, dtype=torch.int32)
        t[:, :2] = table
        outs.append(ops.attention_step(q, k, v, kc.clone(), vc.clone(), t.to(device), lengths))
    # the same scores; 64 roundings of weights and division and a chain of at most 32 / 4 * 4 additions on either side, of what |v| bounds
    assert float((outs[0] - outs[1]).abs().max()) <= 2 * (64 + 32) * U32 * max(float(v.abs().max()), float(vc.abs().max()))


@pytest.mark.gpu
def test_step_over_millions_of_frames():
    """16 million frames that lie on two pages, listed over and over; equal weights, values of one sign."""
    ops = make_ops("cuda:0")
    page, n, hk, d = 1024, 16384 * 1024, 8, 8
    kc = torch.zeros(2, page, hk, d, device="cuda:0")
    vc = equal_terms(2 * page, d, hk).reshape(2, page, hk, d).contiguous().cuda()
    table = torch.zeros(1, n // page + 1, dtype=torch.int32, device="cuda:0")
    table[0, -1] = 1
    q = torch.zeros(1, 1, hk, d, device="cuda:0")
    o = ops.attention_step(q, torch.zeros_like(q), vc[:1, :1].clone(), kc, vc, table, torch.tensor([n], dtype=torch.int32, device="cuda:0"))
    # a wavefront's 32768 frames: blocks of 128 additions, 64 of them; four wavefronts, at most 128 parts; 64 for the weights
    rel = (128 + 64 + 4 + 128 + 64) * U32
    assert float((o.cpu().double() / vc[0, :1].cpu().double() - 1).abs().max()) <= rel


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("side", ["dq", "dk"])
# documents, size of the gradients, of the values, of the keys (queries)
@pytest.mark.parametrize("lens,gs,vs,ks", [([512], 2.0 ** -10, 1.0, 256.0), ([100, 300], 2.0 ** -13, 1.0, 1024.0), ([30, 17], 2.0 ** -13, 0.25, 512.0),
                                           ([40], 1.0, 1.0, 1.0), ([40], 2048.0, 1024.0, 2.0 ** -7), ([5, 20], 2048.0, 1024.0, 2.0 ** -7)])
def test_float16_score_gradients_of_any_size(device, side, lens, gs, vs, ks):
    """Equal weights 1 / n: with q = 0 dq is dS k / 4, with k = 0 dk is dS^T q / 4, dS = (g v - delta) / n between 1e-7 and 1e6."""
    ops = make_ops(device)
    gen = torch.Generator().manual_seed(8)
    n, d = sum(lens), 16
    q, k, v, g = ((torch.randn(n, 1, d, generator=gen) * x).half() for x in (ks, ks, vs, gs))
    (q if side == "dq" else k).zero_()
    plan = ops.attention_plan(lens)
    dev = [x.to(device) for x in (q, k, v)]
    o, lse = ops.attention(plan, *dev)
    got = dict(zip(("dq", "dk", "dv"), ops.attention_backward(plan, g.to(device), *dev, o, lse)))[side].cpu().double()[:, 0]
    u, at = U[torch.float16], 0
    for m in lens:
        s = slice(at, at + m)
        at += m
        Q, K, V, G = (x[s, 0].double() for x in (q, k, v, g))
        dP, O = G @ V.T, V.mean(0)
        delta = (dP / m).sum(1, keepdim=True)
        dS = (dP - delta) / m
        # dS: the weights to 64 roundings; dP a product of 16 terms; delta from the rounded o (dq) or a sum of m; what its two parts lose
        err = 64 * U32 * dS.abs() + (G.abs() @ V.abs().T * 18 * U32 + G.abs() @ O.abs()[:, None] * (u + 18 * U32)
                                    + (dP.abs() / m).sum(1, keepdim=True) * (m + 16) * U32) / m
        err = err + 2.0 ** -38 * (dS.abs().max() if max(lens) <= 32 else dS.abs().amax(1, keepdim=True) if side == "dq" else dS.abs().amax(0, keepdim=True))
        if side == "dq":
            want, e, size = dS @ K / 4, err @ K.abs() / 4, dS.abs() @ K.abs() / 4
        else:
            want, e, size = dS.T @ Q / 4, err.T @ Q.abs() / 4, dS.abs().T @ Q.abs() / 4
        bound = u * want.abs() + (1 + u) * (e + (m / 16 + 16) * U32 * size) + 2.0 ** -25
        assert bool(torch.isfinite(got[s]).all()) and bool(((got[s] - want).abs() <= bound).all()), float(((got[s] - want).abs() / bound).max())


def test_shared_memory_is_found_and_nothing_else():
    """Against a set of the bytes that each of two views of one small buffer addresses."""
    from deepof_amd.attention import _share
    gen = np.random.default_rng(3)
    buf = torch.zeros(300, dtype=torch.float16)
    wide = buf.view(torch.float32)

    def view():
        base, size = (buf, 2) if gen.random() < 0.7 else (wide, 4)
        shape = tuple(int(x) for x in gen.integers(1, 5, 3))
        stride = tuple(int(x) for x in gen.choice([0, 1, 2, 3, 4, 6, 8, 12, 24, 36], 3))
        room = base.numel() - 1 - sum((n - 1) * s for n, s in zip(shape, stride))
        if room < 0:
            return view()
        at = int(gen.integers(0, room + 1))
        t = torch.as_strided(base, shape, stride, at)
        idx = at + sum(s * np.arange(n).reshape([-1 if k == d else 1 for k in range(3)]) for d, (n, s) in enumerate(zip(shape, stride)))
        return t, {int(i) * size + b for i in idx.ravel() for b in range(size)}

    seen = [0, 0]
    for _ in range(3000):
        (a, bytes_a), (b, bytes_b) = view(), view()
        want = bool(bytes_a & bytes_b)
        seen[want] += 1
        assert _share(a, b) == want, (a.shape, a.stride(), a.storage_offset(), b.shape, b.stride(), b.storage_offset())
    assert min(seen) > 300


@pytest.mark.parametrize("device", DEVICES)
def test_slices_of_one_buffer(device):
    """Outputs whose heads or elements lie between those of the inputs are taken; an lse in the output's memory, and caches that
    overlap without beginning together, are not."""
    ops = make_ops(device)
    gen = torch.Generator().manual_seed(6)
    plan = ops.attention_plan([4, 5])
    for buf, at in ((torch.randn(9, 3, 4, 16, generator=gen), lambda b, i: b[:, :, i]), (torch.randn(4, 3, 9, 16, generator=gen), lambda b, i: b[i].transpose(0, 1)),
                    (torch.randn(3, 4, 9, 16, generator=gen), lambda b, i: b[:, i].transpose(0, 1))):
        buf = buf.to(device)
        o, q, k, v = (at(buf, i) for i in range(4))
        want, _ = ops.attention(plan, q.contiguous(), k.contiguous(), v.contiguous())
        got, _ = ops.attention(plan, q, k, v, out=o)
        assert got is o and torch.equal(o, want)
        with pytest.raises(ValueError, match="share memory"):
            ops.attention(plan, q, k, v, out=q)
    q = torch.randn(9, 3, 16, generator=gen).to(device)
    o = torch.zeros(9, 3, 16, device=device)
    with pytest.raises(ValueError, match="share memory"):
        ops.attention(plan, q, q, q, out=o, lse=o.view(-1)[:27].view(9, 3))
    with pytest.raises(ValueError, match="share memory"):
        ops.attention(plan, q, q, q, lse=q.view(-1)[:27].view(9, 3))
    for bad in (dict(lse=q.view(-1)[5]), dict(out=q.view(-1)[5]), dict(lse=torch.zeros((), device=device)), dict(out=torch.zeros((), device=device))):
        with pytest.raises(ValueError):
            ops.attention(plan, q, q, q, **bad)
    kv = torch.randn(6, 8, 4, 16, generator=gen).to(device)
    new, table, lengths = torch.randn(1, 1, 2, 16, device=device), torch.zeros(1, 1, dtype=torch.int32, device=device), torch.zeros(1, dtype=torch.int32, device=device)
    for a, b in ((kv[:4, :, :2], kv[1:5, :, :2]), (kv[:, :, :2], kv[:, :, 1:3])):
        with pytest.raises(ValueError, match="share"):
            ops.attention_step(new, new, new, a, b, table, lengths)
    ops.attention_step(new, new, new, kv[:, :, :2], kv[:, :, 2:], table, lengths)
    assert torch.equal(kv[0, 0], torch.cat((new, new), 2)[0, 0])


def test_launch_limits():
    """Less than 2^32 threads in a launch: counted for the tiles that are launched, at 256 threads for a tall one and 64 for a flat
    one.  Refused before anything is launched; nothing of the (absent) tensors is touched."""
    ops = make_ops("cpu")

    def record(lens, heads):
        off = np.concatenate(([0], np.cumsum(np.asarray(lens, dtype=np.int64))))
        plan = _capi.AttnPlan()
        _capi.check(ops.lib, ops.lib.dof_attn_plan_size(len(lens), off.ctypes.data, off.ctypes.data, 0, C.byref(plan)), "size")
        st = (heads * 64, 64)
        return plan, _capi.PACK_ATTENTION.pack(_capi.DTYPE_BF16, 64, heads, heads, 0.125, 0.0, *(st * 8))

    # one document of 2^29 rows, 2 heads: 2^23 tall tiles are launched, the 2^25 flat ones are not
    plan, rec = record([2 ** 29], 2)
    assert ops._bytes("dof_attention_workspace_bytes", C.byref(plan), rec) >= 2 ** 29 * 2 * 4
    hold = torch.zeros(64)
    some = hold.data_ptr() // 64 * 64 + 64
    for lens, heads in (([2 ** 30] * 2, 1), ([2 ** 30], 4), ([20] * 70000, 1000)):
        plan, rec = record(lens, heads)
        rc = ops.lib.dof_attention_forward(C.byref(plan), some, rec, some, some, some, 0, some, some, 0)
        assert rc < 0 and b"too many tiles" in ops.lib.dof_last_error_string()
        rc = ops.lib.dof_attention_backward(C.byref(plan), some, rec, some, some, some, some, 0, some, some, some, some, some, some, 0)
        assert rc < 0 and b"too many tiles" in ops.lib.dof_last_error_string()


@pytest.mark.parametrize("device", DEVICES)
def test_written_tensors_count_as_changed(device):
    """A graph that saved a tensor which a call then writes over must not run backward on the new values."""
    ops = make_ops(device)
    pos, freqs = torch.arange(6, dtype=torch.int32, device=device), torch.ones(8, dtype=torch.float64, device=device)
    w = torch.ones(6, 2, 16, device=device, requires_grad=True)
    q, k = (torch.randn(6, 2, 16, device=device) for _ in range(2))
    plan = ops.attention_plan([6])
    lse = torch.zeros(6, 2, device=device)
    kc, vc = (torch.zeros(2, 16, 2, 16, device=device) for _ in range(2))
    new = q[None, :1]

    def step():
        ops.attention_step(new, new, new, kc, vc, torch.zeros(1, 1, dtype=torch.int32, device=device), torch.zeros(1, dtype=torch.int32, device=device),
                           out=torch.zeros_like(new))

    for held, call in ((q, lambda: ops.norm_rope(q, k, pos, freqs, q_out=q)), (k, lambda: ops.norm_rope(q, k, pos, freqs, k_out=k)),
                       (k, lambda: ops.attention(plan, q, q, q, out=k)), (lse, lambda: ops.attention(plan, q, q, q, lse=lse)), (kc, step), (vc, step)):
        y = ((w.flatten()[0] if held.shape != w.shape else w) * held).sum()
        call()
        with pytest.raises(RuntimeError, match="inplace operation"):
            y.backward()
    y = (w * q).sum()
    ops.norm_rope(q, k, pos, freqs)  # writes to its own outputs only
    y.backward()
    with torch.inference_mode():
        x = torch.randn(6, 2, 16, device=device)
        ops.norm_rope(x, k, pos, freqs, q_out=x)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("d", [8, 32, 72])
def test_step_with_infinite_keys(device, dtype, d):
    """A cached key whose score is -inf has weight zero, as one whose score is far below the others'."""
    ops = make_ops(device)
    g = torch.Generator().manual_seed(9)
    q, k, v = (torch.randn(1, 1, 2, d, generator=g).to(dtype).to(device) for _ in range(3))
    q[..., 0] = 1.0
    kc, vc = (torch.randn(3, 16, 2, d, generator=g).to(dtype).to(device) for _ in range(2))
    table, lengths = torch.arange(3, dtype=torch.int32, device=device)[None], torch.tensor([40], dtype=torch.int32, device=device)
    outs = []
    for low in (-30000.0, -math.inf):
        kc[0, 3, :, 0], kc[1, 7, 1, 0] = low, low
        outs.append(ops.attention_step(q, k, v, kc, vc.clone(), table, lengths))
    assert bool(torch.isfinite(outs[1]).all()) and torch.equal(*outs)


@pytest.mark.gpu
def test_long_weight_gradients_of_one_sign():
    """33 million rows of equal positive terms (two million tokens of one memory, expanded)."""
    ops = make_ops("cuda:0")
    n, heads, d = 1 << 21, 16, 256
    gen = torch.Generator().manual_seed(14)
    x, g = ((0.5 + torch.rand(1, 1, d, generator=gen)).bfloat16().cuda() for _ in range(2))
    wide = [t.expand(n, heads, d) for t in (x, g)]
    few = [t.expand(n, 1, d) for t in (x, g)]
    w = torch.ones(d, device="cuda:0")
    dwq, dwk = ops.norm_rope_backward(wide[1], few[1], wide[0], few[0], torch.zeros(n, dtype=torch.int32, device="cuda:0"),
                                      torch.zeros(0, dtype=torch.float64, device="cuda:0"), w, w)[2:]
    X, G = x.cpu().double(), g.cpu().double()
    want = (G * X / torch.sqrt((X * X).mean(-1, keepdim=True) + 1e-6))[0, 0] * n
    # a thread's 64 rows of a chunk of 64 tokens, 32 chunks, 2 exchanges and 4 wavefronts, 1024 partial rows in 32 chains of 32; 40 for a term
    rel = (64 + 32 + 6 + 64 + 40) * U32
    assert float((dwq.cpu().double() / (want * heads) - 1).abs().max()) <= rel
    assert float((dwk.cpu().double() / want - 1).abs().max()) <= rel


@pytest.mark.parametrize("device", DEVICES)
def test_float16_log_sum_exp_of_a_lifted_sum(device):
    """The factor of float16 weights leaves the sum before its logarithm: equal scores of 0 over n keys give log n to 4 roundings of
    it (a logarithm good to one step, log 2 and the product with it), not of log(2048 n)."""
    ops = make_ops(device)
    for n in (3, 5, 7, 11, 13):
        q, k = torch.zeros(1, 1, 16, dtype=torch.float16, device=device), torch.zeros(n, 1, 16, dtype=torch.float16, device=device)
        _, lse = ops.attention(ops.attention_plan([1], [n]), q, k, k)
        assert abs(float(lse) - math.log(n)) <= 4 * U32 * math.log(n), n


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES[1:], ids=str)
@pytest.mark.parametrize("n,new", [(300, 1), (1500, 3)])
def test_step_is_as_good_as_rounding_its_result(device, dtype, n, new):
    """16-bit weights keep their rest: o is off by its own rounding and fp32 arithmetic."""
    ops = make_ops(device)
    gen = torch.Generator().manual_seed(15)
    d, page = 64, 100
    q, k, v = (torch.randn(1, new, 2, d, generator=gen).to(dtype) for _ in range(3))
    pages = -(-(n + new) // page)
    kc, vc = (torch.randn(pages, page, 2, d, generator=gen).to(dtype) for _ in range(2))
    table = torch.arange(pages, dtype=torch.int32, device=device)[None]
    o = ops.attention_step(*(x.to(device) for x in (q, k, v)), kc.to(device), vc.to(device), table, torch.tensor([n], dtype=torch.int32, device=device))
    K, V = kc.reshape(-1, 2, d)[:n].double(), vc.reshape(-1, 2, d)[:n].double()
    for t in range(new):
        for h in range(2):
            Kt, Vt = (torch.cat((c[:, h], x[0, :t + 1, h].double())) for c, x in ((K, k), (V, v)))
            Q = q[0, t, h].double()
            p = torch.softmax(Kt @ Q / 8, 0)
            want = p @ Vt
            # scores: chains of 64 / 8 + 8 roundings of |q||k|; twice that and 64 for the weights, 2 u^2 for what value and rest leave
            es = float((Kt.abs() @ Q.abs()).max()) / 8 * 16 * U32
            rel = 2 * es + (64 + n / 32) * U32 + 2 * U[dtype] ** 2
            bound = U[dtype] * want.abs() + 1.01 * rel * (p @ Vt.abs()) + TINY[dtype]
            assert bool(((o[0, t, h].cpu().double() - want).abs() <= bound).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("heads,n", [(8, 32), (64, 32), (16, 25), (48, 200)])
def test_float32_sums_over_many_query_heads(device, heads, n):
    """One key head under many query heads: dv and dk add up the rows of all of them."""
    ops = make_ops(device)
    d = 16
    q, g = (equal_terms(n, d).expand(n, heads, d).contiguous() for _ in range(2))
    k, v = torch.zeros(n, 1, d), torch.zeros(n, 1, d)
    v[:1, 0, 0] = 1.0  # dS: g0 (1 - 1 / n) / n for key 0, - g0 / n^2 for the others
    plan = ops.attention_plan([n])
    args = [x.to(device) for x in (q, k, v)]
    o, lse = ops.attention(plan, *args)
    dq, dk, dv = (x.cpu().double() for x in ops.attention_backward(plan, g.to(device), *args, o, lse))
    # a chain of 256 additions (where each takes one term, as in the emulation), blocks of 256, at most 64 workgroups' parts; 64 for weights
    rel = (256 + heads * n / 256 + 64 + 64) * U32
    assert float((dv / (g[:1, :1].double() * heads) - 1).abs().max()) <= rel
    size = g[0, 0, 0].double() * q[:1, :1].double() * heads * d ** -0.5
    want = torch.cat((size * (1 - 1 / n), (-size / n).expand(n - 1, 1, d)))
    # dS of the other keys is the difference 0 - delta, delta to rel
    assert float((dk / want - 1).abs().max()) <= 3 * rel


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("many,hk,long", [(1500, 1, {3: 1200, 1030: 600, 1499: 900}), (257, 2, {256: 700, 0: 0}), (2, 1100, {0: 1200})])
def test_step_of_many_streams_or_heads(device, many, hk, long):
    """More streams than a workgroup finds parts for, idle ones among them; so many heads that long streams stay whole."""
    ops = make_ops(device)
    d, page = 8, 16
    gen = torch.Generator().manual_seed(17)
    lens = [int(x) for x in torch.randint(0, 40, (many,), generator=gen)]
    for b, n in long.items():
        lens[b] = n
    pages = [-(-(n + 1) // page) for n in lens]
    table, at = torch.full((many, max(pages)), -1, dtype=torch.int32), 0
    for b, c in enumerate(pages):
        table[b, :c] = torch.arange(at, at + c, dtype=torch.int32)
        at += c
    kc, vc = (torch.randn(at, page, hk, d, generator=gen) for _ in range(2))
    q, k, v = (torch.randn(many, 1, hk, d, generator=gen) for _ in range(3))
    lengths = torch.tensor(lens, dtype=torch.int32)
    idle = [b for b in (1, 5, 1100) if b < many]
    lengths[idle] = -1
    kd, vd, out = kc.to(device), vc.to(device), torch.full((many, 1, hk, d), 7.0, device=device)
    ops.attention_step(*(x.to(device) for x in (q, k, v)), kd, vd, table.to(device), lengths.to(device), out=out)
    for b in range(many):
        if b in idle:
            assert bool((out[b] == 7).all())
            continue
        rows = table[b, :pages[b]].long()
        K, V = (torch.cat((c[rows].reshape(-1, hk, d)[:lens[b]], x[b])).double() for c, x in ((kc, k), (vc, v)))
        s = torch.einsum("nhd,hd->hn", K, q[b, 0].double()) * d ** -0.5
        want = torch.einsum("hn,nhd->hd", torch.softmax(s, 1), V)
        es = float((K.abs() * q[b].double().abs()).sum(-1).max()) * d ** -0.5 * 16 * U32  # chains of 8 / 8 + 8 roundings
        bound = (2 * es + (64 + lens[b] / 32) * U32) * float(V.abs().max()) * 1.01
        assert float((out[b, 0].cpu().double() - want).abs().max()) <= bound
        kc[table[b, lens[b] // page], lens[b] % page], vc[table[b, lens[b] // page], lens[b] % page] = k[b, 0], v[b, 0]
    assert torch.equal(kd.cpu(), kc) and torch.equal(vd.cpu(), vc)


@pytest.mark.gpu
def test_graph_of_many_streams_follows_lengths():
    """300 streams, whose parts a kernel of its own lists: replayed while lengths and idle streams change, the eager results."""
    ops = make_ops("cuda:0")
    many, hk, d, page = 300, 2, 16, 16
    gen = torch.Generator().manual_seed(18)
    lens = torch.randint(0, 60, (many,), generator=gen, dtype=torch.int32)
    lens[7], lens[290] = 1500, 900
    table = torch.zeros(many, 100, dtype=torch.int32)
    at = 0
    for b in range(many):
        c = -(-(int(lens[b]) + 8) // page)
        table[b, :c] = torch.arange(at, at + c, dtype=torch.int32)
        at += c
    caches = [torch.randn(at, page, hk, d, generator=gen) for _ in range(2)]
    q, k, v = (torch.randn(many, 1, h, d, generator=gen).cuda() for h in (4, hk, hk))
    (kd, vd), (ke, ve), table = [x.cuda() for x in caches], [x.cuda() for x in caches], table.cuda()
    ln, out = lens.cuda(), torch.zeros_like(q)
    ops.attention_step(q, k, v, kd.clone(), vd.clone(), table, ln, out=out.clone())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attention_step(q, k, v, kd, vd, table, ln, out=out)
    want = out.clone()
    for i in range(4):
        q.mul_(1.1)
        if i == 2:
            ln[[7, 20]] = -1
        le = ln.clone()
        graph.replay()
        torch.cuda.synchronize()
        ops.attention_step(q, k, v, ke, ve, table, le, out=want)
        assert torch.equal(out, want) and torch.equal(kd, ke) and torch.equal(vd, ve)
        ln[ln >= 0] += 1
