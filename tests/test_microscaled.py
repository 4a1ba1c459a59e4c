"""Microscaled rows without a GPU: the plain implementation against itself, and what is refused."""
import numpy as np
import pytest
import torch

from alofa_amd import ops
from alofa_amd.errors import AlofaError
from plain import microscaled as pm


def test_bytes_are_whole_tiles():
    assert ops.MXRows.bytes(1, 1, "e2m1") == 1024 + 64
    assert ops.MXRows.bytes(16, 128, "e4m3") == 2048 + 64
    assert ops.MXRows.bytes(17, 129, "e4m3") == 4 * (2048 + 64)


@pytest.mark.parametrize("rows,k,kind", [(0, 5, "e2m1"), (5, 0, "e4m3"), (-1, 5, "e2m1"), (4, 4, "e5m2"), (4, 4, "")])
def test_sizes_and_kinds_that_are_refused(rows, k, kind):
    with pytest.raises(AlofaError):
        ops.MXRows.bytes(rows, k, kind)


def test_operands_off_the_gpu_are_refused():
    with pytest.raises(AlofaError):
        ops.MXRows(4, 4, "e2m1", buffer=torch.empty(4096, dtype=torch.uint8))
    x = torch.zeros(4, 32)
    for call in (lambda: ops.mx_quantize(x, x), lambda: ops.mx_values(x, x), lambda: ops.mx_from_codes(x.to(torch.uint8), x.to(torch.uint8), 32, "e4m3"),
                 lambda: ops.rmsnorm_mx(x, x, x[0], 1e-6), lambda: ops.gemm_mx(x, x, x), lambda: ops.gemm_mx_shares(x, x, x), lambda: ops.gemm_swiglu_mx(x, x, x, x)):
        with pytest.raises(AlofaError):
            call()


@pytest.mark.parametrize("kind", ["e2m1", "e4m3"])
def test_plain_rounding_is_the_nearest_within_half_a_step(kind):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((40, 77)) * np.exp2(rng.integers(-40, 40, (40, 1)).astype(float))
    e = pm.scale_exponents(x, kind)
    v = pm.rounded(x, kind)
    assert (np.abs(v - x) <= pm.half_step(np.abs(x), e, kind) * (1 + 1e-12)).all()
    grid = pm.GRID[kind]
    s = np.exp2(e.astype(float)).repeat(32, axis=1)[:, :77]
    nearest = np.abs(np.abs(x / s)[..., None] - grid).min(-1)
    assert np.allclose(np.abs(np.abs(x / s) - np.abs(v / s)), nearest, rtol=0, atol=1e-12)
    # (half the scale would be too small for the block's largest magnitude)
    top = np.abs(pm.blocks(x)).max(-1)
    assert (top <= pm.LIMIT[kind] * np.exp2(e.astype(float))).all() and (top > pm.LIMIT[kind] * np.exp2(e - 1.0)).all()


def test_plain_elements_are_torchs():
    codes = np.arange(256)
    want = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    got = pm.values(codes[None], np.full((1, 8), 127, dtype=np.uint8), 256, "e4m3")[0]
    assert np.array_equal(got, want, equal_nan=True)
