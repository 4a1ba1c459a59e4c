"""Microscaled rows without a GPU: the plain implementation against itself, and what is refused."""
import numpy as np
import pytest
import torch

from alofa_amd import ops
from alofa_amd.csrc.build import load
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


# ------------------------------------------------------------- the engine's choice of it

def test_only_layers_that_it_is_built_for(tiny_dirs, tugalix_dirs):
    from alofa_amd.config.registry import load_config
    from alofa_amd.parts.microscaled import KIND, microscaled
    spec = load_config(tiny_dirs["A"]).spec()
    changed = microscaled(spec)
    assert [layer.block.kind for layer in changed.layers] == [KIND] * len(spec.layers) and changed.order == spec.order
    assert [layer.parts for layer in changed.layers] == [layer.parts for layer in spec.layers]
    for d in tugalix_dirs.values():
        with pytest.raises(AlofaError):
            microscaled(load_config(d).spec())


def test_the_model_reads_the_same_tensors(tiny_dirs):
    from alofa_amd.config.registry import load_config
    from alofa_amd.model import expected_tensors
    from alofa_amd.parts.microscaled import microscaled
    spec = load_config(tiny_dirs["C"]).spec()
    assert list(expected_tensors(microscaled(spec)).items()) == list(expected_tensors(spec).items())


@pytest.mark.parametrize("dtype,matrices", [("float32", "mxfp4"), ("bfloat16", "mxfp8"), ("bfloat16", "")])
def test_choices_that_are_refused(tiny_dirs, dtype, matrices):
    from alofa_amd.model import load_model
    with pytest.raises(AlofaError) as e:
        load_model(tiny_dirs["A"], dtype, "cuda:0", matrices)
    assert "matrices" in str(e.value)


@pytest.mark.parametrize("dtype,matrices", [("float32", "mxfp4"), ("bfloat16", "nvfp4")])
def test_the_command_refuses_them_too(tiny_dirs, monkeypatch, dtype, matrices):
    from alofa_amd import cli
    monkeypatch.setenv("ALOFA_WEIGHTS", str(tiny_dirs["A"]))
    monkeypatch.setenv("ALOFA_DTYPE", dtype)
    monkeypatch.setenv("ALOFA_MATRICES", matrices)
    with pytest.raises(AlofaError) as e:
        cli.main(["5,6"])
    assert "ALOFA_MATRICES" in str(e.value)


def test_an_engine_over_a_given_model_does_not_change_its_matrices():
    from alofa_amd import Engine
    with pytest.raises(AlofaError):
        Engine(None, model=(None, None), matrices="mxfp4")


@pytest.mark.parametrize("M,N,K,kind", [(0, 32, 64, "e4m3"), (4, -1, 64, "e4m3"), (4, 32, 0, "e2m1"), (4, 32, 1 << 25, "e2m1"), (1 << 25, 32, 64, "e4m3"), (4, 32, 64, "e5m2")])
def test_shares_of_sizes_and_kinds_that_are_refused(M, N, K, kind):
    with pytest.raises(AlofaError):
        ops.mx_shares(M, N, K, kind)


# ------------------------------------------------------------- what the entries themselves refuse (addresses of nothing: what is not refused asks for a GPU and finds none)

no_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are made up: only for machines on which nothing can be launched")
A, B, C, D = (1 << (44 + i) for i in range(4))      # apart, and aligned


def said(entry, *args):
    """What the entry refuses its arguments with."""
    assert ops._answer(entry, *args) != 0
    return load().alofa_last_error().decode()


@no_gpu
@pytest.mark.parametrize("kind", [0, 4])
@pytest.mark.parametrize("k,threads", [(32, 256), (2048, 256), (2049, 512), (2176, 512), (4096, 512), (4097, 768), (6144, 768), (6145, 1024), (6272, 1024)])
def test_a_norms_launch_has_fewer_than_2_32_threads(k, threads, kind):
    most = ((1 << 32) - 1) // threads

    def norm(rows):
        return said("alofa_rmsnorm_mx", A, kind, B, 0, None, 0, 0, 0, None, 0, C, 1e-6, rows, k, 0)
    assert "than a launch takes" in norm(most + 1) and "no ROCm-capable device" in norm(most)


@no_gpu
@pytest.mark.parametrize("kind", [0, 4])
@pytest.mark.parametrize("kernel", ["stream", "stream64x64", "64x64"])
@pytest.mark.parametrize("M", [1, 20, 70])
def test_the_streaming_kernels_grid_has_room_for_65535_shares(M, kernel, kind):
    def product(shares):
        return said("alofa_gemm_mx", None, ops.F32, 5, shares, A, B, kind, C, None, M, 5, 1 << 24, ops.STORE, ops.MX_FORMS[kernel], 0)
    assert "no ROCm-capable device" in product(65535)
    assert ("no ROCm-capable device" if kernel == "64x64" else "more shares than") in product(65536)


NO_GPU, MEETS = "no ROCm-capable device", "what is written overlaps what is read"


@no_gpu
@pytest.mark.parametrize("kind", ["e2m1", "e4m3"])
def test_what_is_written_may_not_overlap_what_is_read(kind):
    number = ops.MX_KINDS[kind]
    rows, k, n = 40, 256, 256      # (N = K: gated rows would fit the place of the rows they are made of)
    held, matrix = ops.MXRows.bytes(rows, k, kind), ops.MXRows.bytes(n, k, "e2m1")

    def quantise(out, x, ldx=k, dtype=ops.F32):
        return said("alofa_mx_quantize", out, number, x, dtype, ldx, rows, k, 0)

    def values(out, q, ldo=k):
        return said("alofa_mx_values", out, ops.F32, ldo, q, number, rows, k, 0)

    def codes(out, codes, scales):
        return said("alofa_mx_from_codes", out, number, codes, k, scales, k // 32, rows, k, 0)

    def norm(out, x, w, add, total, ldx=k, ld_add=k, ld_total=k, shares=2, stride=rows * k):
        return said("alofa_rmsnorm_mx", out, number, x, ldx, add, shares, stride, ld_add, total, ld_total, w, 1e-6, rows, k, 0)

    def product(out, a, w, bias=None, parts=None, shares=1):
        return said("alofa_gemm_mx", out, ops.F32, n, shares, parts, a, number, w, bias, rows, n, k, ops.STORE, -1, 0)

    def gated(out, a, gate, up):
        return said("alofa_gemm_swiglu_mx", out, number, a, number, gate, up, rows, n, k, 0, -1, 0)
    apart = [quantise(A, B), quantise(A, A + held), quantise(A + rows * k * 4, A), quantise(A + 4 * k, A, 4096),      # (the last two: behind all rows, and in the room between two of them)
             values(A, B), codes(A, B, C), norm(A, B, C, D, B), norm(A, B, C, D, D + 8 * rows * k), norm(A, B, C, D, B + 4 * k, 2 * k, k, 2 * k), norm(A, B, C, B, B + 8 * rows * k), norm(A, B, C, 0, 0, shares=0),
             product(A, B, C), product(A, B, C, D), product(A, B, C, None, D, 2), product(A, A + 4 * rows * n, C), gated(A, B, C, D), gated(A, B, C, C), gated(A, A + held, C, D)]
    meet = [quantise(A, A), quantise(A + 64, A, 4096), quantise(A, A + held - 16), quantise(A + rows * k * 4 - 16, A), values(A, A), values(A + held - 4, A), codes(A, A, B), codes(A, B, A + 16), codes(A, A + held - 1, B),
            norm(A, A, B, C, C + 8 * rows * k), norm(A, B, C, D, A), norm(A, B, A, C, D), norm(A, B, C, D, D), norm(A, B, C, D, D + 4 * rows * k), norm(A, B, C, A + 16, D), norm(A, B, C, D, C + 16 - 4 * k),
            norm(A, B, C, D, B + 4), norm(A, B, C, D, B + 4 * k, 2 * k, k, 3 * k), norm(A, B, C, D, B, 0), norm(A, B, C, D, B + 4 * k - 16, 2 * k, k, 2 * k), norm(A, A, B, 0, 0, shares=0),
            product(A, A, C), product(A, B, A), product(A, B, C, A), product(A, B, C, None, A, 2), product(A, B, C, None, B, 2), product(None, B, C, None, C + matrix - 16, 2), product(A + held - 4, A, C),
            gated(A, A, B, C), gated(A, B, A, C), gated(A, B, C, A), gated(A + held - 16, A, B, C), gated(A, B, A + held - 16, C), gated(A + matrix - 16, B, C, A)]
    for i, s in enumerate(apart):
        assert NO_GPU in s, (i, s)
    for i, s in enumerate(meet):
        assert MEETS in s, (i, s)
