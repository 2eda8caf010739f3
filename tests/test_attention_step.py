"""attention_step (new frames against a paged cache) against the formulas in 64 bits; pages, idle streams, refusals; and the three
operators as they are used together."""
import math

import numpy as np
import pytest
import torch

from deepof_amd.attention import rotary_frequencies
from sequence_common import DEVICES, DTYPES, TINY, U, U32, assert_within, draw, make_ops


def reference(t, table, lengths, page, n_pages, cap, slopes, dtype, kc, vc):
    """64-bit o with its bound (as in the attention tests: weights rounded once to the type, scores a chain of head_dim products)
    and the caches after the call."""
    u = U[dtype]
    low = u if dtype != torch.float32 else 0.0
    q, k, v = (t[n].double() for n in "qkv")
    b, new, hq, d = q.shape
    hk = k.shape[2]
    kc, vc = kc.clone(), vc.clone()
    o, bound = torch.zeros_like(q), torch.zeros_like(q)
    for s in range(b):
        length = int(lengths[s])
        if length < 0:
            continue
        cap_rows = table.shape[1] * page
        length = min(length, cap_rows)
        where = []
        for p in range(min(length + new, cap_rows)):
            pg = int(table[s, p // page])
            if 0 <= pg < n_pages:
                if p >= length:
                    kc[pg, p % page], vc[pg, p % page] = t["k"][s, p - length], t["v"][s, p - length]
                where.append((p, pg, p % page))
        pos = torch.tensor([w[0] for w in where])
        K = torch.stack([kc[pg, at] for _, pg, at in where]).double() if where else torch.zeros(0, hk, d, dtype=torch.float64)
        V = torch.stack([vc[pg, at] for _, pg, at in where]).double() if where else torch.zeros(0, hk, d, dtype=torch.float64)
        for i in range(new):
            seen = pos <= length + i if where else torch.zeros(0, dtype=torch.bool)
            for h in range(hq):
                Kh, Vh = K[seen, h // (hq // hk)], V[seen, h // (hq // hk)]
                if len(Kh) == 0:
                    continue
                raw = Kh @ q[s, i, h] * d ** -0.5
                es = (Kh.abs() @ q[s, i, h].abs()) * d ** -0.5 * (d / 8 + 8) * U32
                z = raw
                if cap:
                    z = cap * torch.tanh(raw / cap)
                    es = es + cap * 2.0 ** -21
                if slopes is not None:
                    dist = slopes[h].double() * (length + i - pos[seen])
                    z = z - dist
                    es = es + dist * 2 * U32
                e = float((es + 4 * U32 * z.abs() + 8 * U32).max())
                p = torch.softmax(z, 0)
                o[s, i, h] = p @ Vh
                bound[s, i, h] = u * o[s, i, h].abs() + (1 + u) * (low + 2 * e + 64 * U32) * (p @ Vh.abs()) + TINY[dtype]
    return o, bound, kc, vc


# lengths, new frames, query heads, key heads, head size, page size, cap, bias
CASES = [
    ([0], 1, 1, 1, 8, 1, 0.0, False),
    ([0, 31, 32, 33], 1, 4, 2, 64, 16, 0.0, True),
    ([300, 5], 1, 8, 1, 128, 16, 0.0, False),
    ([70, 290], 3, 8, 2, 96, 100, 6.0, False),
    ([45], 5, 16, 1, 32, 7, 0.0, True),          # 80 rows: three blocks of 32
    ([600], 2, 6, 2, 80, 64, 0.0, False),        # the length in parts
    ([128, 17, 255], 16, 2, 1, 24, 32, 0.0, False),
]


def build(case, dtype, device, seed=0, spare=2):
    lens, new, hq, hk, d, page, cap, bias = case
    g = torch.Generator().manual_seed(seed)
    b = len(lens)
    t = dict(q=draw((b, new, hq, d), dtype, g), k=draw((b, new, hk, d), dtype, g), v=draw((b, new, hk, d), dtype, g))
    pages = [-(-(n + new) // page) for n in lens]
    total = sum(pages) + spare
    order = torch.randperm(total, generator=g).tolist()
    table = torch.full((b, max(pages) + 1), -7, dtype=torch.int32)  # entries behind a stream's pages are never valid
    for s, c in enumerate(pages):
        table[s, :c] = torch.tensor([order.pop() for _ in range(c)], dtype=torch.int32)
    kc, vc = draw((total, page, hk, d), dtype, g), draw((total, page, hk, d), dtype, g)
    slopes = torch.rand(hq, generator=g) * 0.1 if bias else None
    return t, table, torch.tensor(lens, dtype=torch.int32), kc, vc, slopes


def run(ops, t, table, lengths, kc, vc, slopes, cap, device, **kw):
    kd, vd = kc.to(device), vc.to(device)
    o = ops.attention_step(t["q"].to(device), t["k"].to(device), t["v"].to(device), kd, vd, table.to(device), lengths.to(device), cap=cap,
                           slopes=slopes.to(device) if slopes is not None else None, **kw)
    return o, kd.cpu(), vd.cpu()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("case", CASES, ids=str)
def test_step(device, dtype, case):
    ops = make_ops(device)
    t, table, lengths, kc, vc, slopes = build(case, dtype, device)
    o, kd, vd = run(ops, t, table, lengths, kc, vc, slopes, case[6], device)
    want, bound, kw, vw = reference(t, table, lengths, case[5], kc.shape[0], case[6], slopes, dtype, kc, vc)
    assert_within("o", o, want, bound)
    assert torch.equal(kd, kw) and torch.equal(vd, vw)


@pytest.mark.parametrize("device", DEVICES)
def test_more_streams_than_threads(device):
    """300 streams on pages of 5, the long one at 280 in parts, some idle."""
    ops = make_ops(device)
    lens = [(7 * s) % 11 for s in range(300)]
    lens[280] = 700
    case = (lens, 1, 2, 1, 16, 5, 0.0, False)
    t, table, lengths, kc, vc, slopes = build(case, torch.float32, device)
    lengths[3], lengths[299] = -1, -1
    out = torch.full((300, 1, 2, 16), 7.0, device=device)
    o, kd, vd = run(ops, t, table, lengths, kc, vc, slopes, 0.0, device, out=out)
    want, bound, kw, vw = reference(t, table, lengths, 5, kc.shape[0], 0.0, None, torch.float32, kc, vc)
    live = lengths >= 0
    assert_within("o", o.cpu()[live], want[live], bound[live])
    assert bool((o.cpu()[~live] == 7).all()) and torch.equal(kd, kw) and torch.equal(vd, vw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("case", [([20011, 3], 1, 8, 2, 128, 16, 0.0, False), ([9000] * 3 + [40] * 30, 2, 4, 4, 64, 32, 10.0, True)],
                         ids=["long", "ragged"])
def test_step_long(dtype, case):
    ops = make_ops("cuda:0")
    t, table, lengths, kc, vc, slopes = build(case, dtype, "cuda:0", seed=4)
    o, kd, vd = run(ops, t, table, lengths, kc, vc, slopes, case[6], "cuda:0")
    want, bound, kw, vw = reference(t, table, lengths, case[5], kc.shape[0], case[6], slopes, dtype, kc, vc)
    assert_within("o", o, want, bound)
    assert torch.equal(kd, kw) and torch.equal(vd, vw)


@pytest.mark.parametrize("device", DEVICES)
def test_untrusted_device_data(device):
    """Idle streams, lengths behind the table, page indices that the cache does not have."""
    ops = make_ops(device)
    case = ([70, 40, 60, 50], 2, 2, 1, 32, 16, 0.0, False)
    dtype = torch.bfloat16
    t, table, lengths, kc, vc, slopes = build(case, dtype, device)
    lengths[0] = -1
    table[1, 1] = kc.shape[0]        # frames 16 .. 31 are nowhere
    table[2, :] = table[2, :].clone()
    table[3, 3] = -5                 # the new frames have no page: 50, 51 are on the fourth
    lengths[2] = 5000                # behind the table: clamped to its width, nothing is stored
    table[2, -1] = table[2, 0]
    out = torch.full((4, 2, 2, 32), 7.0, dtype=dtype, device=device)
    o, kd, vd = run(ops, t, table, lengths, kc, vc, slopes, 0.0, device, out=out)
    assert o is out and bool((out[0] == 7).all())
    want, bound, kw, vw = reference(t, table, lengths, 16, kc.shape[0], 0.0, None, dtype, kc, vc)
    assert_within("o", o[1:], want[1:], bound[1:])
    assert torch.equal(kd, kw) and torch.equal(vd, vw)
    # a stream without any valid page sees nothing: zeros
    table[1, :] = -1
    o, kd, vd = run(ops, t, table, lengths, kc, vc, slopes, 0.0, device, out=out)
    assert bool((o[1] == 0).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_unseen_places_reach_nothing(device, bad):
    """What lies behind a stream's last frame on its page, on other pages, and a later new frame's values."""
    ops = make_ops(device)
    case = ([37], 3, 2, 1, 32, 16, 0.0, False)
    t, table, lengths, kc, vc, slopes = build(case, torch.float32, device)
    want, _, _ = run(ops, t, table, lengths, kc, vc, slopes, 0.0, device)
    used = [int(x) for x in table[0, :3]]
    kb, vb = torch.full_like(kc, bad), torch.full_like(vc, bad)
    for p in range(37):
        kb[used[p // 16], p % 16], vb[used[p // 16], p % 16] = kc[used[p // 16], p % 16], vc[used[p // 16], p % 16]
    got, _, _ = run(ops, t, table, lengths, kb, vb, slopes, 0.0, device)
    assert torch.equal(got, want)
    t2 = {n: x.clone() for n, x in t.items()}
    t2["k"][0, 2], t2["v"][0, 2] = bad, bad
    got, _, _ = run(ops, t2, table, lengths, kc, vc, slopes, 0.0, device)
    assert torch.equal(got[:, :2], want[:, :2]) and not bool(torch.isfinite(got[:, 2]).any())
    vb = vc.clone()  # a cached frame on the new frames' page: every row sees it
    vb[used[2], 3] = bad
    got, _, _ = run(ops, t, table, lengths, kc, vb, slopes, 0.0, device)
    assert not bool(torch.isfinite(got).any())


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    from deepof_amd._capi import DofError
    ops = make_ops(device)
    case = ([20, 9], 2, 4, 2, 16, 8, 0.0, False)
    t, table, lengths, kc, vc, slopes = build(case, torch.float32, device)
    q, k, v, kc, vc, tb, ln = (x.to(device) for x in (t["q"], t["k"], t["v"], kc, vc, table, lengths))
    for args in ((q.double(), k, v, kc, vc, tb, ln), (q, k[:1], v, kc, vc, tb, ln), (q, k, v[..., :8], kc, vc, tb, ln),
                 (q, k, v, kc.half(), vc, tb, ln), (q, k, v, kc[:, :, :1], vc[:, :, :1], tb, ln), (q, k, v, kc, vc[1:], tb, ln),
                 (q, k, v, kc, vc, tb.long(), ln), (q, k, v, kc, vc, tb[:1], ln), (q, k, v, kc, vc, tb, ln.long()),
                 (q, k, v, kc, vc, tb, ln[:1]), (q[:, :, :3], k, v, kc, vc, tb, ln), (q[0], k, v, kc, vc, tb, ln),
                 (q, k, v, kc[:1].expand(9, 8, 2, 16), kc[:1].expand(9, 8, 2, 16), tb, ln)):
        with pytest.raises(ValueError):
            ops.attention_step(*args)
    with pytest.raises(ValueError, match="two tensors"):
        ops.attention_step(q, k, v, kc, kc, tb, ln)
    with pytest.raises(ValueError, match="share memory"):
        ops.attention_step(q, k, v, kc, vc, tb, ln, out=q)
    with pytest.raises(DofError, match="new frames"):
        ops.attention_step(q[:, :1].expand(2, 17, 4, 16), k[:, :1].expand(2, 17, 2, 16), v[:, :1].expand(2, 17, 2, 16), kc, vc, tb, ln)
    with pytest.raises(DofError, match="head_dim"):
        ops.attention_step(q[..., :4], k[..., :4], v[..., :4], kc[..., :4], vc[..., :4], tb, ln)
    with pytest.raises(DofError):
        ops.attention_step(q, k, v, kc, vc, tb, ln, cap=-1.0)
    with pytest.raises(DofError, match="bad cache"):
        ops.attention_step(q, k, v, kc, vc, tb[:, :0], ln)
    assert ops.attention_step(q[:0], k[:0], v[:0], kc, vc, tb[:0], ln[:0]).shape == (0, 2, 4, 16)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_together(device, dtype):
    """A recording through norm_rope and causal attention at once, and the same frames one by one (then three at a time) through
    norm_rope and attention_step on a paged cache: the same outputs."""
    ops = make_ops(device)
    n, hq, hk, d, page = 75, 4, 2, 32, 16
    g = torch.Generator().manual_seed(11)
    qkv = draw((n, hq + 2 * hk, d), dtype, g).to(device)
    w = [(1.0 + 0.1 * torch.randn(d, generator=g)).to(device) for _ in range(2)]
    freqs = rotary_frequencies(d // 2, device=device)
    slopes = (torch.rand(hq, generator=g) * 0.05).to(device)
    pos = torch.arange(n, dtype=torch.int32, device=device)
    kw = dict(q_weight=w[0], k_weight=w[1])
    q, k = ops.norm_rope(qkv[:, :hq], qkv[:, hq:hq + hk], pos, freqs, **kw)
    v = qkv[:, hq + hk:]
    whole, _ = ops.attention(ops.attention_plan([n], causal=True), q, k, v, slopes=slopes)

    kc, vc = (torch.full((6, page, hk, d), float("nan"), dtype=dtype, device=device) for _ in range(2))
    table = torch.tensor([[4, 0, 5, 2, 1]], dtype=torch.int32, device=device)
    at, outs = 0, []
    while at < n:
        step = 1 if at < 66 else 3
        rows = slice(at, at + step)
        qs, ks = ops.norm_rope(qkv[rows, :hq], qkv[rows, hq:hq + hk], pos[rows], freqs, **kw)
        assert torch.equal(qs, q[rows]) and torch.equal(ks, k[rows])
        outs.append(ops.attention_step(qs[None], ks[None], v[rows][None], kc, vc, table, pos[at:at + 1], slopes=slopes)[0])
        at += step
    # both are within half a step of their own rounding and one rounding of the weights (bound by the largest |v|) of the same numbers
    vmax = float(v.abs().max())
    bound = torch.full(whole.shape, (2 * U[dtype] * 2 + 2.0 ** -17) * vmax, dtype=torch.float64)
    assert_within("frames one by one", torch.cat(outs), whole.cpu().double(), bound)
    assert torch.equal(kc[4], k[:16]) and torch.equal(vc[1, :11], v[64:])


@pytest.mark.gpu
def test_graph_replay_follows_lengths():
    """One captured step, replayed while the caller advances the lengths on the device: the eager results, every time."""
    ops = make_ops("cuda:0")
    case = ([500, 1200, 7], 1, 8, 2, 64, 16, 0.0, False)
    t, table, lengths, kc, vc, slopes = build(case, torch.bfloat16, "cuda:0", spare=6)
    table[table < 0] = 0
    q, k, v, tb, ln = (x.cuda() for x in (t["q"], t["k"], t["v"], table, lengths))
    kd, vd, ke, ve = kc.cuda(), vc.cuda(), kc.cuda(), vc.cuda()
    ops.attention_step(q, k, v, kd, vd, tb, ln)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.attention_step(q, k, v, kd, vd, tb, ln)
        ln.add_(1)
    le = lengths.cuda()
    for i in range(3):
        q.mul_(1.1)
        graph.replay()
        torch.cuda.synchronize()
        want = ops.attention_step(q, k, v, ke, ve, tb, le)
        le += 1
        assert torch.equal(out, want) and torch.equal(kd, ke) and torch.equal(vd, ve) and torch.equal(ln, le)
