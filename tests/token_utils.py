"""Shared by the tests of the token-model operators: unit roundings and element-wise bounds."""
import torch

U32 = 2.0 ** -24                                       # half a float32 step, relative


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def assert_within(got, want, bound, what=""):
    """|got - want| <= bound element by element (want, bound in float64); non-finite values must agree."""
    got, want = got.detach().double().cpu(), want.double().cpu()
    bound = torch.as_tensor(bound, dtype=torch.float64).cpu().expand_as(want)
    fine = torch.isfinite(want)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), f"{what}: infinities differ"
    off = (got - want).abs() - bound
    off[~fine] = 0
    if off.numel():
        at = int(off.argmax())
        assert off.max() <= 0, f"{what}: at {at} got {got.flatten()[at]}, want {want.flatten()[at]}, bound {bound.flatten()[at]}"


def devices():
    import pytest
    return [pytest.param("cpu"), pytest.param("cuda:0", marks=pytest.mark.gpu)]
