"""Edges of the sequence operators: long tails of a softmax, long sums, what a row must not see, memory they may not touch, limits.
Every bound is derived where it stands; u is half a step of the type, relative to the value."""
import math

import pytest
import torch

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
