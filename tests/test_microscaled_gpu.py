"""Microscaled rows on the GPU: every operator against plain numpy in 64 bits, at the sizes, values and layouts where it could go wrong."""
import functools

import numpy as np
import pytest
import torch

from alofa_amd import ops
from alofa_amd.errors import AlofaError
from plain import microscaled as pm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
KINDS = ["e2m1", "e4m3"]
SIZES = [(1, 1), (1, 31), (2, 32), (3, 33), (16, 128), (17, 129), (5, 897), (33, 640), (130, 1000)]


def numbers(rows, k, seed, spread=20):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, k)) * np.exp2(rng.integers(-spread, spread + 1, (rows, -(-k // 32))).astype(float)).repeat(32, axis=1)[:, :k]
    return x.astype(np.float32)


def on(x, dtype=torch.float32):
    return torch.from_numpy(np.ascontiguousarray(x)).to(DEV, dtype)


def strided(x, dtype, by):
    """x on the GPU as the left columns of wider rows (by: further columns) that hold 7."""
    wide = torch.full((x.shape[0], x.shape[1] + by), 7.0, dtype=dtype, device=DEV)
    wide[:, :x.shape[1]] = on(x, dtype)
    return wide[:, :x.shape[1]]


def made(x, kind):
    """x (float32 numpy) as microscaled rows on the GPU, in a buffer whose every byte was 255 before (what is not written shows)."""
    q = ops.MXRows(*x.shape, kind, DEV)
    q.buffer.fill_(255)
    ops.mx_quantize(q, on(x))
    return q


def read(q, dtype=torch.float32):
    out = torch.empty(q.rows, q.k, dtype=dtype, device=DEV)
    ops.mx_values(out, q)
    return out.double().cpu().numpy()


def same(got, want):
    assert np.array_equal(got, want, equal_nan=True), f"{(got != want).sum()} of {got.size} differ, first at {np.argwhere(~((got == want) | (np.isnan(got) & np.isnan(want))))[:3].tolist()}"


# ------------------------------------------------------------- numbers to rows and back

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,k", SIZES)
def test_quantise(rows, k, dtype, kind):
    x = on(numbers(rows, k, rows + k), dtype).double().cpu().numpy()
    for by in (0, 8, 3):      # (rows that 16-byte loads can read, and rows that they cannot)
        q = ops.MXRows(rows, k, kind, DEV)
        q.buffer.fill_(255)
        ops.mx_quantize(q, strided(x.astype(np.float32), dtype, by))
        same(read(q), pm.rounded(x, kind))


@pytest.mark.parametrize("kind", KINDS)
def test_quantise_special_blocks(kind):
    lim, big = pm.LIMIT[kind], np.float32(3.4028235e38)
    grid = pm.GRID[kind]
    ties = np.concatenate([(grid[1:] + grid[:-1]) / 2, -(grid[1:] + grid[:-1]) / 2, [grid[-1]]])
    ties = np.concatenate([ties, np.full(-len(ties) % 31, grid[-1])])
    ties = np.concatenate([np.append(t, grid[-1]) for t in ties.reshape(-1, 31)])      # (every block has the largest element: its scale is 1)
    special = [np.zeros(32), np.full(32, -0.0), np.append(np.zeros(31), lim), np.append(np.zeros(31), np.nextafter(np.float32(lim), np.float32(1e9))), np.append(np.ones(31), -lim),
               np.full(32, 1e-45), np.full(32, 1.17549435e-38), np.linspace(-3e-39, 3e-39, 32), np.full(32, big), np.append(np.full(31, 1.0), big), np.linspace(-1, 1, 32) * 2.0 ** -126,
               np.append(np.full(31, 1.0), np.inf), np.append(np.full(31, 1.0), -np.inf), np.append(np.full(31, 1.0), np.nan), np.full(32, np.nan), np.append(np.zeros(31), 1e-45), ties]
    x = np.concatenate(special).astype(np.float32)[None]
    with np.errstate(over="ignore"):      # (the largest floats round to 2^128, which as a float is infinite)
        same(read(made(x, kind)), pm.rounded(x.astype(np.float64), kind).astype(np.float32).astype(np.float64))


@pytest.mark.parametrize("kind", KINDS)
def test_values_in_bfloat16_and_strided(kind):
    x = numbers(19, 203, 5)
    q = made(x, kind)
    want = torch.from_numpy(pm.rounded(x.astype(np.float64), kind)).bfloat16().double().numpy()
    same(read(q, torch.bfloat16), want)
    for dtype, by in ((torch.bfloat16, 8), (torch.float32, 5)):
        out = strided(np.zeros((19, 203), np.float32), dtype, by)
        ops.mx_values(out, q)
        same(out.double().cpu().numpy(), want)
        assert (out._base[:, 203:] == 7).all()      # (columns beside the values stay as they were)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,k", SIZES)
def test_from_codes(rows, k, kind):
    rng = np.random.default_rng(k)
    scales = rng.integers(90, 160, (rows, -(-k // 32))).astype(np.uint8)
    scales.flat[::7] = 0
    scales.flat[3::11] = 255
    scales.flat[5::13] = 254 if kind == "e2m1" else 200
    code = rng.integers(0, 16 if kind == "e2m1" else 256, (rows, 32 * scales.shape[1]))
    held = code[:, :k + k % 2] if kind == "e2m1" else code[:, :k]      # (the half byte behind an odd row's last number holds something)
    if kind == "e2m1":
        held = held[:, 0::2] | held[:, 1::2] << 4
    for by in (0, 3):
        codes_d = strided(held.astype(np.float32), torch.uint8, by)
        q = ops.mx_from_codes(codes_d, strided(scales.astype(np.float32), torch.uint8, by), k, kind)
        with np.errstate(over="ignore"):
            same(read(q), pm.values(code, scales, k, kind).astype(np.float32).astype(np.float64))


# ------------------------------------------------------------- the norm between sub-layers

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,k,shares", [(1, 1, 0), (1, 33, 1), (3, 896, 0), (8, 896, 1), (5, 1000, 3), (17, 2048, 2), (70, 1536, 1), (130, 129, 4), (4, 5120, 2), (2, 8192, 1), (3, 9000, 2), (3, 27648, 0), (600, 640, 1)])
def test_norm(rows, k, shares, kind):
    x, w = numbers(rows, k, k, 2), numbers(1, k, k + 1, 0)[0]
    add = [numbers(rows, k, k + 2 + s, 2) for s in range(shares)]
    total = x
    if shares:
        sum_ = add[0]
        for a in add[1:]:
            sum_ = sum_ + a
        total = x + sum_
    want = pm.rounded(pm.norm(total.astype(np.float64), w.astype(np.float64), 1e-6), kind)
    for by, in_place in ((0, False), (3, True), (8, True)):
        q = ops.MXRows(rows, k, kind, DEV)
        q.buffer.fill_(255)
        xd = strided(x, torch.float32, by)
        if shares:
            t = xd if in_place else torch.empty(rows, k, device=DEV)
            parts = on(np.stack(add))
            ops.rmsnorm_mx(q, xd, on(w), 1e-6, add=parts if shares > 1 else parts[0], total=t)
            same(t.double().cpu().numpy(), total.astype(np.float64))
            assert in_place or (xd == on(x)).all()
            assert by == 0 or (xd._base[:, k:] == 7).all()
        else:
            ops.rmsnorm_mx(q, xd, on(w), 1e-6)
        same(read(q), want)      # (squares and scaling in 64 bits on both sides: elements differ only where a value lies within 1e-14 of a middle)


def test_norm_rows_that_are_zero_or_not_finite_keep_to_themselves():
    x = numbers(6, 96, 1, 2)
    x[1], x[2, 5], x[3, 7], x[4] = 0.0, np.inf, np.nan, 1e-30
    q = ops.MXRows(6, 96, "e4m3", DEV)
    w = np.ones(96, np.float32)
    ops.rmsnorm_mx(q, on(x), on(w), 1e-6)
    got = read(q)
    ok = [0, 1, 4, 5]
    same(got[ok], pm.rounded(pm.norm(x[ok].astype(np.float64), 1.0, 1e-6), "e4m3"))
    # (an infinity: its own block is NaN, inf / inf, the others are zeros; a NaN takes its whole row along)
    assert np.isnan(got[2, :32]).all() and (got[2, 32:] == 0).all() and np.isnan(got[3]).all()


def test_norm_of_very_large_and_very_small_rows():
    x, w = numbers(6, 896, 3, 2), numbers(1, 896, 4, 0)[0]
    x[1:3] *= np.float32(1e37)      # (squares beyond a float)
    x[3:5] *= np.float32(1e-37)
    w[:10] *= np.float32(1e30)
    want = pm.rounded(pm.norm(x.astype(np.float64), w.astype(np.float64), 1e-6), "e4m3")
    q = ops.MXRows(6, 896, "e4m3", DEV)
    ops.rmsnorm_mx(q, on(x), on(w), 1e-6)
    # (a scale is 2^-127 at least and an element 2^-9: what is below half of that is zero on both sides; below 2^-149 a float has no bits left)
    got = read(q)
    same(got, want.astype(np.float32).astype(np.float64))


@pytest.mark.parametrize("k", [896, 5120])
def test_norm_of_a_row_does_not_depend_on_the_others(k):
    x, w = numbers(300, k, 9, 2), numbers(1, k, 10, 0)[0]
    all_of = ops.MXRows(300, k, "e4m3", DEV)
    ops.rmsnorm_mx(all_of, on(x), on(w), 1e-6)
    one = ops.MXRows(1, k, "e4m3", DEV)
    for r in (0, 15, 16, 299):
        ops.rmsnorm_mx(one, on(x[r:r + 1]), on(w), 1e-6)
        same(read(one)[0], read(all_of)[r])


# ------------------------------------------------------------- products

def operands(M, N, K, kind, seed):
    """Microscaled rows and a matrix on the GPU and the values they stand for."""
    a, w = numbers(M, K, seed, 2), numbers(N, K, seed + 1, 2)
    return made(a, kind), made(w, "e2m1"), pm.rounded(a.astype(np.float64), kind), pm.rounded(w.astype(np.float64), "e2m1")


def off_by(a, w):
    """How far a float32 sum of these products may be off: the products of elements and scales are exact, and an addend meets at most 128 additions within a tile of K, one
    per tile behind it and sixteen more where parts of K meet, each off by 2^-23 of what is there by then at most (2^-24 where it rounds to the nearest)."""
    return (128 + -(-a.shape[1] // 128) + 16) * 2.0 ** -23 * (np.abs(a) @ np.abs(w).T)


PRODUCTS = [(1, 1, 1), (1, 16, 32), (2, 50, 128), (5, 33, 100), (8, 1152, 896), (16, 130, 257), (17, 64, 640), (31, 100, 1500), (33, 48, 129), (48, 257, 896), (64, 96, 4864), (65, 131, 300),
            (130, 300, 1000), (200, 129, 2048), (257, 512, 384), (300, 1000, 513), (515, 260, 896), (1030, 700, 260)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_product(M, N, K, kind):
    a, w, av, wv = operands(M, N, K, kind, M + N + K)
    want, off = av @ wv.T, off_by(av, wv)
    bias, old = numbers(1, N, 3, 3)[0], numbers(M, N, 4, 3)
    for by in (0, 4, 3):
        for dtype in (torch.float32, torch.bfloat16):
            step = 2.0 ** -24 if dtype is torch.float32 else 2.0 ** -8
            out = strided(old, dtype, by)
            ops.gemm_mx(out, a, w, on(bias))
            ref = want + bias
            assert (np.abs(out.double().cpu().numpy() - ref) <= off + 2.0 ** -23 * np.abs(ref) + step * (np.abs(ref) + off)).all()
            assert by == 0 or (out._base[:, N:] == 7).all()
            out = strided(old, dtype, by)
            ops.gemm_mx(out, a, w)
            assert (np.abs(out.double().cpu().numpy() - want) <= off + step * (np.abs(want) + off)).all()
        out = strided(old, torch.float32, by)
        ops.gemm_mx(out, a, w, add_to_out=True)
        ref = want + old
        assert (np.abs(out.double().cpu().numpy() - ref) <= off + 2.0 ** -24 * (np.abs(ref) + off)).all()
        assert by == 0 or (out._base[:, N:] == 7).all()


def check_gated(out, av, gv, uv, act, out_kind):
    M, N = out.rows, out.k
    got = read(out)
    gate, up = av @ gv.T, av @ uv.T
    f = getattr(pm, "silu" if act == "silu" else act)(gate)
    y = f * up
    # the activations' slopes are at most 1.13; exponential, division and product in float32: some ten roundings, those of the exponent weighted with it (|2 c z| below 2^7 here)
    dy = 1.13 * off_by(av, gv) * (np.abs(up) + off_by(av, uv)) + np.abs(f) * off_by(av, uv) + 2.0 ** -15 * np.abs(y)
    # a sum that is off may take a block's scale over a border: half a step of the larger one then
    e = np.maximum(pm.scale_exponents(np.abs(y) + dy, out_kind), pm.scale_exponents(y, out_kind))
    assert (np.abs(got - y) <= dy + pm.half_step(np.abs(y) + dy, e, out_kind) * (1 + 1e-12)).all()
    assert (got == pm.rounded(y, out_kind)).mean() > 0.98 or got.size < 64
    # what the rows are filled up with is zeros: a product over all of them is the product over N
    ones = made(np.ones((1, N), np.float32), "e2m1")
    sums = torch.empty(M, 1, device=DEV)
    ops.gemm_mx(sums, out, ones)
    one = np.ones((1, N))
    assert (np.abs(sums.double().cpu().numpy() - got @ one.T) <= off_by(got, one)).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("M,N,K", [(5, 40, 256), (300, 200, 384)])
def test_products_of_blocks_with_scales_far_apart(M, N, K, kind):
    rng = np.random.default_rng(K)
    blocks = K // 32
    ea, ew = rng.integers(0, 251, (M, blocks)), rng.integers(-20, 21, (N, blocks))
    ca = rng.integers(0, 16 if kind == "e2m1" else 256, (M, K))
    if kind == "e4m3":
        ca = np.where((ca & 127) == 127, 0, ca)      # (no NaN)
    cw = rng.integers(0, 16, (N, K))
    # rows' scales from end to end of the range, the matrix's so that every block's products come out around 2^0
    ea = np.broadcast_to(rng.integers(2, 249, (1, blocks)), (M, blocks)) + rng.integers(-2, 3, (M, blocks))
    ew = np.clip(254 - ea[:1] + ew, 0, 254)
    pairs = lambda c: c[:, 0::2] | c[:, 1::2] << 4      # noqa: E731
    to = lambda c: torch.from_numpy(np.ascontiguousarray(c.astype(np.uint8))).to(DEV)      # noqa: E731
    a = ops.mx_from_codes(to(pairs(ca) if kind == "e2m1" else ca), to(ea), K, kind)
    w = ops.mx_from_codes(to(pairs(cw)), to(ew), K)
    av, wv = pm.values(ca, ea, K, kind), pm.values(cw, ew, K, "e2m1")
    out = torch.empty(M, N, device=DEV)
    ops.gemm_mx(out, a, w)
    assert (np.abs(out.double().cpu().numpy() - av @ wv.T) <= off_by(av, wv)).all()


def test_matrices_beyond_32_bits_of_bytes():
    """The last rows of 2.4 GB of matrix, and of rows as long, against the same tiles as matrices of their own."""
    N, K = 1_100_007, 4096
    g = torch.Generator(DEV).manual_seed(1)

    def tail(q, tiles):      # the last row tiles of q as rows of their own
        per = -(-K // 128) * (1024 if q.kind == "e2m1" else 2048)
        rows = q.rows - (-(-q.rows // 16) - tiles) * 16
        t = ops.MXRows(rows, K, q.kind, DEV)
        all_tiles, scales = -(-q.rows // 16), -(-K // 128) * 64
        t.buffer[:tiles * per] = q.buffer[(all_tiles - tiles) * per:all_tiles * per]
        t.buffer[tiles * per:tiles * (per + scales)] = q.buffer[all_tiles * per + (all_tiles - tiles) * scales:all_tiles * (per + scales)]
        return t

    w = ops.MXRows(N, K, "e2m1", DEV)
    assert w.buffer.numel() > 1 << 31
    w.buffer.random_(0, 256, generator=g)
    w.buffer[-(-N // 16) * 32 * 1024:].random_(110, 130, generator=g)
    small = tail(w, 4)
    for M, kernel in ((3, "stream"), (70, "64x64"), (70, "256x128")):
        a = made(numbers(M, K, M, 1), "e4m3")
        out = torch.empty(M, N, dtype=torch.bfloat16, device=DEV)
        ops.gemm_mx(out, a, w, kernel=kernel)
        part = torch.empty(M, small.rows, dtype=torch.bfloat16, device=DEV)
        ops.gemm_mx(part, a, small, kernel=kernel)
        assert torch.equal(out[:, -small.rows:], part) and out.isfinite().all()
        del out
    # rows: 4.6 GB of numbers in, 2.4 GB of elements; and as many rows of a product
    out = torch.empty(N, K, dtype=torch.bfloat16, device=DEV)
    ops.mx_values(out, w)
    part = torch.empty(small.rows, K, dtype=torch.bfloat16, device=DEV)
    ops.mx_values(part, small)
    assert torch.equal(out[-small.rows:], part)
    again = ops.MXRows(N, K, "e2m1", DEV)
    ops.mx_quantize(again, out)
    part2 = torch.empty_like(part)
    ops.mx_values(part2, tail(again, 4))
    assert torch.equal(part2, part)      # (values of the format stay as they are)
    narrow = made(numbers(130, K, 9, 1), "e2m1")
    prod = torch.empty(N, 130, device=DEV)
    ops.gemm_mx(prod, w, narrow)
    few = torch.empty(small.rows, 130, device=DEV)
    ops.gemm_mx(few, small, narrow, kernel="256x128")
    assert (prod[-small.rows:] - few).abs().max() <= 1e-4 * few.abs().max()


FORMS = [f for f in ops.MX_FORMS if f is not None]


@pytest.mark.parametrize("kernel", FORMS)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (3, 40, 130), (70, 290, 1100), (300, 530, 384), (513, 260, 257)])
def test_every_kernel_takes_every_product(M, N, K, kind, kernel):
    a, w, av, wv = operands(M, N, K, kind, M + N + K)
    want, off = av @ wv.T, off_by(av, wv)
    for by in (0, 3):
        out = strided(numbers(M, N, 4, 3), torch.float32, by)
        ops.gemm_mx(out, a, w, kernel=kernel)
        assert (np.abs(out.double().cpu().numpy() - want) <= off).all()
        assert by == 0 or (out._base[:, N:] == 7).all()
    tiles = -(-K // 128)
    for shares in {1, min(3, tiles), tiles}:
        parts = torch.full((shares, M, N), 7.0, device=DEV)
        ops.gemm_mx_shares(parts, a, w, kernel=kernel)
        assert (np.abs(parts.double().sum(0).cpu().numpy() - want) <= off).all()


@pytest.mark.parametrize("kernel", [f for f in FORMS if f not in ("256x160", "stream64x64")])      # (the first's columns do not go in pairs of gate and up)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("out_kind", KINDS)
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (3, 40, 130), (70, 290, 300), (300, 530, 384), (513, 130, 257)])
def test_every_kernel_takes_every_gated_product(M, N, K, out_kind, kind, kernel):
    a, g, u = numbers(M, K, 1, 1), numbers(N, K, 2, 1) * np.float32(2 / np.sqrt(K)), numbers(N, K, 3, 1) * np.float32(1 / np.sqrt(K))
    av, gv, uv = pm.rounded(a.astype(np.float64), kind), pm.rounded(g.astype(np.float64), "e2m1"), pm.rounded(u.astype(np.float64), "e2m1")
    out = ops.MXRows(M, N, out_kind, DEV)
    out.buffer.fill_(255)
    ops.gemm_swiglu_mx(out, made(a, kind), made(g, "e2m1"), made(u, "e2m1"), kernel=kernel)
    check_gated(out, av, gv, uv, "silu", out_kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("M,N,K,shares", [(1, 33, 129, 2), (8, 896, 4864, 3), (40, 130, 1000, 8), (130, 512, 2048, 2), (300, 640, 1152, 9)])
def test_shares_add_up(M, N, K, shares, kind):
    a, w, av, wv = operands(M, N, K, kind, M + N + K)
    parts = torch.full((shares, M, N), 7.0, device=DEV)
    ops.gemm_mx_shares(parts, a, w)
    edges = [-(-K // 128) * s // shares * 128 for s in range(shares + 1)]
    for s in range(shares):
        at = slice(edges[s], min(edges[s + 1], K))
        assert (np.abs(parts[s].double().cpu().numpy() - av[:, at] @ wv[:, at].T) <= off_by(av[:, at], wv[:, at])).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("M", [3, 40, 200, 600])
def test_rows_that_are_not_finite_keep_to_themselves(M, kind):
    a = numbers(M, 300, 1, 2)
    a[1, 40], a[2, 299] = np.nan, np.inf
    w = numbers(200, 300, 2, 2)
    w[5, 0] = np.inf
    out = torch.empty(M, 200, device=DEV)
    ops.gemm_mx(out, made(a, kind), made(w, "e2m1"))
    bad = ~np.isfinite(out.cpu().numpy())
    want = np.zeros((M, 200), bool)
    want[1], want[2], want[:, 5] = True, True, True
    assert (bad == want).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("out_kind", KINDS)
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 32, 64), (2, 57, 130), (8, 4864, 896), (17, 200, 300), (33, 129, 1000), (64, 300, 257), (130, 260, 640), (300, 700, 300), (515, 384, 896)])
def test_gated(M, N, K, act, out_kind, kind):
    # (gates of some units, so that the activation bends)
    a, g, u = (numbers(r, K, M + N + i, 1) * s for i, (r, s) in enumerate(((M, 1.0), (N, 2.0 / np.sqrt(K)), (N, 1.0 / np.sqrt(K)))))
    av, gv, uv = pm.rounded(a.astype(np.float64), kind), pm.rounded(g.astype(np.float64), "e2m1"), pm.rounded(u.astype(np.float64), "e2m1")
    out = ops.MXRows(M, N, out_kind, DEV)
    out.buffer.fill_(255)
    ops.gemm_swiglu_mx(out, made(a, kind), made(g, "e2m1"), made(u, "e2m1"), act)
    check_gated(out, av, gv, uv, act, out_kind)


# ------------------------------------------------------------- as they are used together

def chain(x, attn, mats, norm_w, bias):
    """The second half of a layer: output product in shares, norm of the stream, gate and up, down. Returns the stream and what the products of the way were given."""
    T, h = x.shape
    q = ops.MXRows(T, attn.shape[1], "e4m3", DEV)
    ops.mx_quantize(q, attn)
    parts = torch.empty(2, T, h, device=DEV)
    ops.gemm_mx_shares(parts, q, mats["o"])
    normed = ops.MXRows(T, h, "e4m3", DEV)
    ops.rmsnorm_mx(normed, x, norm_w, 1e-6, add=parts, total=x)
    act = ops.MXRows(T, mats["gate"].rows, "e4m3", DEV)
    ops.gemm_swiglu_mx(act, normed, mats["gate"], mats["up"])
    ops.gemm_mx(x, act, mats["down"], add_to_out=True)
    qkv = torch.empty(T, mats["qkv"].rows, dtype=torch.bfloat16, device=DEV)
    ops.gemm_mx(qkv, normed, mats["qkv"], bias)
    return x, qkv


def chain_operands(T, seed):
    h, d, ff, n = 320, 256, 720, 384
    sizes = {"o": (h, d), "gate": (ff, h), "up": (ff, h), "down": (h, ff), "qkv": (n, h)}
    w = {name: numbers(*s, seed + i, 0) / np.float32(np.sqrt(s[1])) for i, (name, s) in enumerate(sizes.items())}
    return numbers(T, h, seed + 10, 1), on(numbers(T, d, seed + 11, 1), torch.bfloat16), w, 1 + numbers(1, h, seed + 12, 0)[0] / 4, numbers(1, n, seed + 13, 0)[0]


@pytest.mark.parametrize("T", [1, 9, 70, 300])
def test_half_a_layer(T):
    x, attn, w, norm_w, bias = chain_operands(T, 50)
    mats = {n: made(m, "e2m1") for n, m in w.items()}
    got, qkv = chain(on(x), attn, mats, on(norm_w), on(bias))
    # step by step in 64 bits, roundings to the formats at their places: what differs is an element here and there that a last bit takes to its neighbour (half a step of e4m3 is 2^-4)
    v = {n: pm.rounded(m.astype(np.float64), "e2m1") for n, m in w.items()}
    t = x + pm.rounded(attn.double().cpu().numpy(), "e4m3") @ v["o"].T
    n = pm.rounded(pm.norm(t, norm_w.astype(np.float64), 1e-6), "e4m3")
    a = pm.rounded(pm.silu(n @ v["gate"].T) * (n @ v["up"].T), "e4m3")
    out, want_qkv = t + a @ v["down"].T, n @ v["qkv"].T + bias
    for g, r, step in ((got, out, 2.0 ** -24), (qkv, want_qkv, 2.0 ** -8)):
        off = np.linalg.norm(g.double().cpu().numpy() - r) / np.linalg.norm(r)
        assert off <= step + 2.0 ** -4 * 2.0 ** -4, off      # (were a part in 256 of all elements a whole step off: far more than last bits can move)


@pytest.mark.parametrize("T", [1, 9, 70, 300])
def test_captured_and_replayed(T):
    x, attn, w, norm_w, bias = chain_operands(T, 80)
    mats = {n: made(m, "e2m1") for n, m in w.items()}
    norm_w, bias = on(norm_w), on(bias)
    xs, attns = on(x), attn.clone()
    chain(xs, attns, mats, norm_w, bias)      # (once before the capture)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out, qkv = chain(xs, attns, mats, norm_w, bias)
    for i in range(4):
        xi, ai = numbers(T, 320, 200 + i, 1), on(numbers(T, 256, 300 + i, 1), torch.bfloat16)
        want, want_qkv = chain(on(xi), ai, mats, norm_w, bias)
        xs.copy_(on(xi)), attns.copy_(ai)
        graph.replay()
        assert torch.equal(out, want) and torch.equal(qkv, want_qkv)
        torch.cuda.synchronize()


def test_without_the_binding_the_results_are_the_same(monkeypatch):
    from alofa_amd.csrc import calls
    x, attn, w, norm_w, bias = chain_operands(9, 50)
    mats = {n: made(m, "e2m1") for n, m in w.items()}
    want, want_qkv = chain(on(x), attn, mats, on(norm_w), on(bias))
    monkeypatch.setattr(ops, "_binding", calls)
    got, qkv = chain(on(x), attn, mats, on(norm_w), on(bias))
    assert torch.equal(got, want) and torch.equal(qkv, want_qkv)
    test_refusals()


def test_two_streams_at_once():
    jobs = []
    for i, T in enumerate((5, 300)):
        x, attn, w, norm_w, bias = chain_operands(T, 20 * i)
        jobs.append((x, attn, {n: made(m, "e2m1") for n, m in w.items()}, on(norm_w), on(bias), torch.cuda.Stream()))
    want = [chain(on(x), *rest)[0].clone() for x, *rest, _ in jobs]
    for _ in range(3):
        got = []
        starts = [on(x) for x, *_ in jobs]
        torch.cuda.synchronize()
        for x, (_, *rest, stream) in zip(starts, jobs):
            with torch.cuda.stream(stream):
                got.append(chain(x, *rest)[0])
        torch.cuda.synchronize()
        for g, r in zip(got, want):
            assert torch.equal(g, r)


# ------------------------------------------------------------- what is refused

def test_refusals():
    a, w = made(numbers(4, 64, 1), "e4m3"), made(numbers(32, 64, 2), "e2m1")
    x = torch.zeros(4, 64, device=DEV)
    out = torch.zeros(4, 32, device=DEV)
    weight = torch.ones(64, device=DEV)
    act = ops.MXRows(4, 32, "e4m3", DEV)
    bad = [lambda: ops.MXRows(4, 64, "e4m3", buffer=torch.empty(100, dtype=torch.uint8, device=DEV)),
           lambda: ops.MXRows(4, 64, "e4m3", buffer=torch.empty(8192, dtype=torch.uint8, device=DEV)[1:]),
           lambda: ops.MXRows(4, 64, "e4m3", buffer=torch.empty(8192, dtype=torch.int8, device=DEV)),
           lambda: ops.mx_quantize(a, x[:3]), lambda: ops.mx_quantize(a, x.half()), lambda: ops.mx_quantize(a, x.t()), lambda: ops.mx_quantize(x, x), lambda: ops.mx_quantize(a, x.cpu()),
           lambda: ops.mx_values(x[:, :63], a), lambda: ops.mx_values(x.double(), a), lambda: ops.mx_values(x[:1].expand(4, 64), a), lambda: ops.mx_values(x, x),
           lambda: ops.mx_from_codes(torch.zeros(4, 64, dtype=torch.uint8, device=DEV), torch.zeros(4, 2, dtype=torch.uint8, device=DEV), 64, "e2m1"),
           lambda: ops.mx_from_codes(torch.zeros(4, 32, dtype=torch.uint8, device=DEV), torch.zeros(4, 3, dtype=torch.uint8, device=DEV), 64, "e2m1"),
           lambda: ops.mx_from_codes(torch.zeros(4, 64, dtype=torch.uint8, device=DEV), torch.zeros(4, 2, dtype=torch.uint8, device=DEV), 64, "e2m3"),
           lambda: ops.mx_from_codes(torch.zeros(5, 64, dtype=torch.uint8, device=DEV), torch.zeros(5, 2, dtype=torch.uint8, device=DEV), 64, "e4m3", out=a),
           lambda: ops.rmsnorm_mx(a, x, weight[:32], 1e-6), lambda: ops.rmsnorm_mx(a, x, weight, 0.0), lambda: ops.rmsnorm_mx(a, x, weight, float("nan")), lambda: ops.rmsnorm_mx(a, x.bfloat16(), weight, 1e-6),
           lambda: ops.rmsnorm_mx(a, x, weight, 1e-6, add=x), lambda: ops.rmsnorm_mx(a, x, weight, 1e-6, total=x), lambda: ops.rmsnorm_mx(a, x, weight, 1e-6, add=x[:2], total=x),
           lambda: ops.rmsnorm_mx(a, x, weight, 1e-6, add=x.bfloat16(), total=x), lambda: ops.rmsnorm_mx(a, x, weight, 1e-6, add=x, total=x[:1].expand(4, 64)),
           lambda: ops.gemm_mx(out, a, a), lambda: ops.gemm_mx(out, w, a), lambda: ops.gemm_mx(out[:, :31], a, w), lambda: ops.gemm_mx(out.half(), a, w), lambda: ops.gemm_mx(out, x, w),
           lambda: ops.gemm_mx(out, a, w, weight), lambda: ops.gemm_mx(out.bfloat16(), a, w, add_to_out=True), lambda: ops.gemm_mx(out, a, w, torch.zeros(32, device=DEV), add_to_out=True),
           lambda: ops.gemm_mx(out, made(numbers(4, 65, 1), "e4m3"), w), lambda: ops.gemm_mx(out[:1].expand(4, 32), a, w),
           lambda: ops.gemm_mx_shares(torch.zeros(2, 4, 32, device=DEV), a, w), lambda: ops.gemm_mx_shares(torch.zeros(0, 4, 32, device=DEV), a, w), lambda: ops.gemm_mx_shares(out, a, w),
           lambda: ops.gemm_swiglu_mx(act, a, w, made(numbers(31, 64, 2), "e2m1")), lambda: ops.gemm_swiglu_mx(act, a, w, a), lambda: ops.gemm_swiglu_mx(a, a, w, w),
           lambda: ops.gemm_swiglu_mx(act, a, w, w, "relu"), lambda: ops.gemm_swiglu_mx(out, a, w, w),
           lambda: ops.gemm_mx(out, a, w, kernel="rows"), lambda: ops.gemm_mx_shares(torch.zeros(1, 4, 32, device=DEV), a, w, kernel="tiles512"), lambda: ops.gemm_swiglu_mx(act, a, w, w, kernel="tiled"),
           lambda: ops.gemm_swiglu_mx(act, a, w, w, kernel="256x160")]
    for k, call in enumerate(bad):
        with pytest.raises(AlofaError):
            call()
            pytest.fail(f"call {k} was not refused")
    ops.gemm_mx(out, a, w)      # (and what is left as it was still runs)
    torch.cuda.synchronize()


def test_more_rows_than_a_norms_launch_takes_are_refused():
    rows = 1 << 24      # (a block of 256 threads each: 2^32 threads)
    out = ops.MXRows(rows, 32, "e2m1", DEV)
    out.buffer[:64].zero_()
    with pytest.raises(AlofaError):
        ops.rmsnorm_mx(out, torch.ones(1, 32, device=DEV).expand(rows, 32), torch.ones(32, device=DEV), 1e-6)
    torch.cuda.synchronize()
    assert not out.buffer[:64].any()


@pytest.mark.parametrize("kernel", ["256x160", "stream64x64"])
def test_forms_that_gated_products_do_not_have_are_refused(kernel):
    a, w, out = made(numbers(40, 64, 1), "e4m3"), made(numbers(32, 64, 2), "e2m1"), ops.MXRows(40, 32, "e4m3", DEV)
    out.buffer.fill_(7)
    with pytest.raises(AlofaError):
        ops.gemm_swiglu_mx(out, a, w, w, kernel=kernel)
    torch.cuda.synchronize()
    assert (out.buffer == 7).all()


@pytest.mark.parametrize("kernel", FORMS)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("M,N,K,shares", [(3, 40, 260, 3), (70, 290, 1100, 4), (300, 136, 900, 8)])
def test_every_kernel_takes_shares(M, N, K, shares, kind, kernel):
    a, w, av, wv = operands(M, N, K, kind, M + K)
    parts = torch.full((shares, M, N), float("nan"), device=DEV)
    ops.gemm_mx_shares(parts, a, w, kernel=kernel)
    tiles, got = -(-K // 128), parts.double().cpu().numpy()
    for s in range(shares):
        cut = slice(128 * (tiles * s // shares), 128 * (tiles * (s + 1) // shares))
        assert (np.abs(got[s] - av[:, cut] @ wv[:, cut].T) <= off_by(av[:, cut], wv[:, cut])).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("k", [96, 896, 2500, 9000])
def test_norm_beyond_the_largest_float(k, kind):
    """Weights so large that rows come out beyond 2^128: elements of their own as far as scales go, NaN behind that. Read by a product with 2^-20 times the identity, whose outputs fit a float."""
    x, w = numbers(6, k, 21, 0), numbers(1, k, 22, 0)[0]
    x[1, 1:], x[2, 2:], x[5] = 0, 0, 0      # (a number alone in its row: the root of k times its weight)
    w[:40] *= np.float32(1e38)
    w[:3] = 3e38, -3e38, 2.0 ** 100
    w[64:70] = 3.4028235e38, 1e-38, -1.0, 3.4e38, 1e34, 0.0
    y = pm.norm(x.astype(np.float64), w.astype(np.float64), 1e-6)
    assert (np.abs(y) >= 2.0 ** 128).any()
    want = pm.rounded(y, kind)
    q = ops.MXRows(6, k, kind, DEV)
    q.buffer.fill_(255)
    ops.rmsnorm_mx(q, on(x), on(w), 1e-6)
    out = torch.empty(6, k, device=DEV)
    ops.gemm_mx(out, q, made(np.eye(k, dtype=np.float32) * np.float32(2.0 ** -20), "e2m1"))
    got, bad = out.double().cpu().numpy(), np.isnan(want).any(1)
    assert not bad.all() and np.isnan(got[bad]).all()      # (a NaN takes its row of the product along)
    same(got[~bad], want[~bad] * 2.0 ** -20)
    with np.errstate(over="ignore"):      # (beyond 2^128 a float is infinite)
        same(read(q), want.astype(np.float32).astype(np.float64))


def test_gated_products_in_the_place_of_their_rows_are_refused():
    a, w = made(numbers(40, 64, 1), "e4m3"), made(numbers(64, 64, 2), "e2m1")
    before = a.buffer.clone()
    for out in (a, ops.MXRows(40, 64, "e4m3", buffer=a.buffer), ops.MXRows(40, 64, "e2m1", buffer=a.buffer[1024:])):
        with pytest.raises(AlofaError, match="overlaps"):
            ops.gemm_swiglu_mx(out, a, w, w)
    torch.cuda.synchronize()
    assert torch.equal(a.buffer, before)


def test_the_sum_in_columns_beside_the_stream():
    wide = on(numbers(40, 512, 1, 1))
    x, w, add = wide[:, :256], on(numbers(1, 256, 2, 1)[0]), on(numbers(40, 256, 3, 1))
    q, r, total = ops.MXRows(40, 256, "e4m3", DEV), ops.MXRows(40, 256, "e4m3", DEV), wide[:, 256:]
    want, stream = torch.empty(40, 256, device=DEV), x.clone()
    ops.rmsnorm_mx(q, x, w, 1e-6, add=add, total=want)
    ops.rmsnorm_mx(r, x, w, 1e-6, add=add, total=total)
    assert torch.equal(total, want) and torch.equal(x, stream)
    same(read(r), read(q))


SHARED_OUT = [(40, 97, 8192, "e4m3"), (20, 64, 9001, "e4m3"), (300, 66, 8200, "e4m3")] + [(*s, kind) for kind in KINDS for s in ((1, 7, 40000), (5, 33, 40000), (33, 131, 16385), (130, 50, 12000), (64, 96, 16384))]


@pytest.mark.parametrize("M,N,K,kind", SHARED_OUT)
def test_products_whose_sum_the_rule_shares_out(M, N, K, kind):
    """Shares of K that a launch of its own adds up, with every epilogue."""
    shares = ops._answer("alofa_gemm_mx_shares", M, N, K, ops.MX_KINDS[kind], 0)
    assert shares > 1
    a, w, av, wv = operands(M, N, K, kind, M + N + K)
    want, off = av @ wv.T, off_by(av, wv)
    bias, old = numbers(1, N, 3, 3)[0], numbers(M, N, 4, 3)
    asked = []

    def scratch(name, shape, dtype):
        asked.append(shape)
        return torch.full(shape, float("nan"), dtype=dtype, device=DEV)
    for by in (0, 8, 3):
        for dtype in (torch.float32, torch.bfloat16):
            step = 2.0 ** -24 if dtype is torch.float32 else 2.0 ** -8
            for b in (None, bias):
                out = strided(old, dtype, by)
                ops.gemm_mx(out, a, w, None if b is None else on(b), scratch=scratch)
                ref = want if b is None else want + b
                assert (np.abs(out.double().cpu().numpy() - ref) <= off + 2.0 ** -23 * np.abs(ref) + step * (np.abs(ref) + off)).all()
                assert by == 0 or (out._base[:, N:] == 7).all()
        out = strided(old, torch.float32, by)
        ops.gemm_mx(out, a, w, add_to_out=True)
        ref = want + old
        assert (np.abs(out.double().cpu().numpy() - ref) <= off + 2.0 ** -24 * (np.abs(ref) + off)).all()
        assert by == 0 or (out._base[:, N:] == 7).all()
    assert asked == [(shares * M * N,)] * 12


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,k,shares", [(1, 40, 2), (5, 896, 3), (17, 2176, 2), (6, 1000, 4), (3, 9000, 2)])
def test_norm_of_shares_and_rows_that_lie_apart_or_are_one_and_the_same(rows, k, shares, kind):
    """Shares in wider rows, at distances of their own, one share or one row many times over; a weight and a stream at any address."""
    x, w = numbers(rows, k, 5, 2), numbers(1, k, 6, 0)[0]
    add = np.stack([numbers(rows, k, 7 + s, 2) for s in range(shares)])

    def check(xd, wd, parts, xv=x, addv=add):
        total = xv + functools.reduce(np.add, addv)
        q, t = ops.MXRows(rows, k, kind, DEV), torch.empty(rows, k, device=DEV)
        q.buffer.fill_(255)
        ops.rmsnorm_mx(q, xd, wd, 1e-6, add=parts, total=t)
        same(t.double().cpu().numpy(), total.astype(np.float64))
        same(read(q), pm.rounded(pm.norm(total.astype(np.float64), w.astype(np.float64), 1e-6), kind))
    xd, wd, ad = on(x), on(w), on(add)
    for rows_by, k_by in ((0, 8), (2, 0), (3, 4), (1, 3)):      # (rows and columns between the shares)
        room = torch.full((shares, rows + rows_by, k + k_by), float("nan"), device=DEV)
        room[:, :rows, :k] = ad
        check(xd, wd, room[:, :rows, :k])
    by_row = torch.full((rows, shares, k), float("nan"), device=DEV)      # (the shares of a row side by side)
    by_row.copy_(ad.transpose(0, 1))
    check(xd, wd, by_row.transpose(0, 1))
    check(xd, wd, ad[:1].expand(shares, rows, k), addv=add[:1].repeat(shares, 0))
    check(xd, wd, ad[:, :1].expand(shares, rows, k), addv=add[:, :1].repeat(rows, 1))
    check(xd, wd, ad[0].expand(shares, rows, k), addv=add[:1].repeat(shares, 0))
    check(xd[:1].expand(rows, k), wd, ad, xv=x[:1].repeat(rows, 0))
    check(xd, wd, xd.expand(shares, rows, k), addv=x[None].repeat(shares, 0))      # (what is added may be the stream)
    odd = torch.empty(k + 1, device=DEV)[1:]
    odd.copy_(wd)
    assert odd.data_ptr() % 16 == 4
    check(xd, odd, ad)
    at = torch.empty(rows * k + 1, device=DEV)[1:].view(rows, k)
    at.copy_(xd)
    check(at, wd, ad)
