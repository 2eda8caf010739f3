"""Shared pieces of the sequence-operator tests: the operators on the emulated build (CPU) or on the device, plain 64-bit forms of
their definitions, and elementwise error bounds.

Bounds count roundings: ``U[dtype]`` is half a unit in the last place relative to the value (the output's own rounding), ``U32`` the
same for the fp32 arithmetic in between."""
import pytest
import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
U32 = 2.0 ** -24
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}  # what a subnormal result may lose
DEVICES = [pytest.param("cpu", id="emu"), pytest.param("cuda:0", id="gpu", marks=pytest.mark.gpu)]
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def make_ops(device):
    if device == "cpu":
        from deepof_amd.attention import AttentionOps
        from emu_util import emu_lib
        return AttentionOps(emu_lib(), "cpu")
    from deepof_amd.attention import create_attention_ops
    return create_attention_ops(device)


def draw(shape, dtype, gen, std=1.0):
    return (torch.randn(shape, generator=gen, dtype=torch.float64) * std).to(dtype)


def strided(t, device, how):
    """The same values on the device in another memory order: 'plain', 'packed' (heads inside a wider row), 'head_major' (the
    rows of a head side by side), 'odd' (rows and start at odd element offsets: no wide access is aligned)."""
    r, h, d = t.shape
    if how == "plain":
        return t.to(device).contiguous()
    if how == "packed":
        buf = torch.full((r, h + 3, d), float("nan"), dtype=t.dtype, device=device)
        view = buf[:, 2:2 + h]
    elif how == "head_major":
        view = torch.full((h, r, d), float("nan"), dtype=t.dtype, device=device).transpose(0, 1)
    else:
        buf = torch.full((r * (h * d + 3) + 1,), float("nan"), dtype=t.dtype, device=device)
        view = torch.as_strided(buf, (r, h, d), (h * d + 3, d, 1), 1)
    view.copy_(t.to(device))
    return view


def assert_within(name, got, want, bound):
    got, want, bound = got.detach().cpu().double(), want.cpu(), bound.cpu()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert torch.isfinite(got).all(), f"{name}: not finite"
    over = (got - want).abs() - bound
    assert (over <= 0).all(), (f"{name}: error {float((got - want).abs().flatten()[over.argmax()]):.3e} over bound "
                               f"{float(bound.flatten()[over.argmax()]):.3e} at value {float(want.flatten()[over.argmax()]):.3e}")
