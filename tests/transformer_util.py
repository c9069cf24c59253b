"""Shared by the tests of the transformer operators: devices, types, tolerances.

A rounding to a type is off by at most half a step, eps / 2 of the value.  The
fp32 arithmetic in front of it is counted in units of U = 2^-24.
"""

import pytest
import torch

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):
    """The rounding of numbers under the least normal one: half of the least step."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def assert_within(got, want, tolerance, what=""):
    """|got - want| <= tolerance, element by element; all in fp64."""
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    tolerance = torch.as_tensor(tolerance, dtype=torch.float64).detach().cpu().expand_as(want)
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} for {tuple(want.shape)}"
    over = (got - want).abs() - tolerance
    bad = ~(over <= 0)
    if bad.any():
        i = int(torch.where(bad, torch.nan_to_num(over, nan=1e30), -1e30).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, worst at {i}: got {got.flatten()[i].item():.9g}, "
                             f"want {want.flatten()[i].item():.9g}, tolerance {tolerance.flatten()[i].item():.3g}")


def replays(make, rounds=3):
    """Captures make() (after a warm run on the side) and yields its outputs after
    every replay, with eager work and a synchronisation in between."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        make()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = make()
    for _ in range(rounds):
        graph.replay()
        torch.cuda.synchronize()
        yield out
        (torch.randn(512, 512, device="cuda") @ torch.randn(512, 512, device="cuda")).sum().item()
