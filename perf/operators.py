"""Microscaled operators as the engine runs them: rows and matrices in blocks of 32 values of 4 or 8 bits with one power of two per block.

A value is an element times its block's scale. Elements: "e2m1" (magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6) or "e4m3" (up to 448); a scale is one byte
e + 127 for 2^e. The scale of a block is the smallest power of two under which its largest magnitude is at most half a step beyond the largest
element (7 for e2m1, 464 for e4m3), never below 2^-127; elements are rounded to the nearest, ties to the even one. Matrices are held as e2m1.

Kinds of case (every size is in the case itself):

  quantise  ``rows`` x ``k`` numbers of ``dtype`` to ``kind`` (and the values that these stand for)
  norm      total = x + (add[0] + add[1] + ...) over ``shares`` parts, RMSNorm of total, to ``kind``: the stream between two sub-layers
  product   ``rows`` bfloat16 rows to ``kind``, times a matrix [n, k] of e2m1; ``to``: "store" (bias, bfloat16 out) or "add" (to the float32 stream)
  gated     ``rows`` bfloat16 rows to ``kind``, silu(x gate^T) * (x up^T) to ``kind``: the first half of a feed-forward"""
import math

import torch

own = False

DEVICE = "cuda:0"
LIMIT = {"e2m1": 7.0, "e4m3": 464.0}      # the largest magnitude of a block under its scale
SMALLEST = {"e2m1": (0, 1), "e4m3": (-6, 3)}      # exponent of the smallest normal element, bits behind the point
LARGEST = {"e2m1": 6.0, "e4m3": 448.0}
EPS = 1e-6


def listed():
    def quantise(name, rows, k, dtype, kind):
        return {"name": name, "do": "quantise", "rows": rows, "k": k, "dtype": dtype, "kind": kind}

    def norm(name, rows, k, shares, kind):
        return {"name": name, "do": "norm", "rows": rows, "k": k, "shares": shares, "kind": kind}

    def product(name, rows, n, k, to, kind):
        return {"name": name, "do": "product", "rows": rows, "n": n, "k": k, "to": to, "kind": kind}

    def gated(name, rows, n, k, kind):
        return {"name": name, "do": "gated", "rows": rows, "n": n, "k": k, "kind": kind}
    return [
        # what attention leaves for eight requests that decode, on its way to the output matrix
        quantise("quantise 8 x 896", 8, 896, "bfloat16", "e4m3"),
        # a feed-forward matrix as it is loaded
        quantise("matrix 18944 x 3584", 18944, 3584, "bfloat16", "e2m1"),
        # one user who waits for each token
        norm("norm 1 x 896", 1, 896, 1, "e4m3"),
        # a full batch that decodes at a large width, behind a product whose sum was shared out
        norm("norm 64 x 5120", 64, 5120, 4, "e4m3"),
        # a tick's prompt tokens
        norm("norm 2048 x 3584", 2048, 3584, 1, "e4m3"),
        # queries, keys and values of one token: the smallest product
        product("product 1, 1152 x 896", 1, 1152, 896, "store", "e4m3"),
        # decoding where the matrix is what a step reads
        product("product 32, 3584 x 18944", 32, 3584, 18944, "add", "e4m3"),
        # a short prompt: rows that fill no tile
        product("product 333, 4608 x 3584", 333, 4608, 3584, "store", "e4m3"),
        # a tick's prompt tokens through the largest matrix
        product("product 2048, 5120 x 27648", 2048, 5120, 27648, "add", "e4m3"),
        # the same with activations of four bits
        product("product 2048, 18944 x 3584 4-bit", 2048, 18944, 3584, "store", "e2m1"),
        # eight requests that decode
        gated("gated 8, 4864 x 896", 8, 4864, 896, "e4m3"),
        # prompt tokens, no whole number of tiles
        gated("gated 1500, 18944 x 3584", 1500, 18944, 3584, "e4m3"),
    ]


def draw(rng):
    def between(lo, hi):      # spread over the logarithm
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    widths = [896, 1536, 2048, 3584, 5120]

    def width():      # a configuration's, or any
        return rng.choice(widths) if rng.random() < 0.5 else between(33, 5120)
    do, kind = rng.choice(["quantise", "norm", "product", "product", "gated"]), rng.choice(["e4m3", "e4m3", "e2m1"])
    if do == "quantise":
        k = width()
        return {"do": do, "rows": between(1, max(2, 60000000 // k)), "k": k, "dtype": rng.choice(["bfloat16", "float32"]), "kind": kind}
    if do == "norm":
        return {"do": do, "rows": between(1, 2048), "k": width(), "shares": rng.choice([1, 1, 2, 3, 4]), "kind": kind}
    k, n = width(), between(48, 18944)
    if do == "product":
        if rng.random() < 0.3:
            n, k = k, n
        return {"do": do, "rows": between(1, 2048), "n": n, "k": k, "to": rng.choice(["store", "add"]), "kind": kind}
    return {"do": do, "rows": between(1, 1200), "n": n, "k": k, "kind": kind}


# ------------------------------------------------------------------ the plain form

def _exponents(x):
    """floor(log2 |x|) of numbers (0 for zero)."""
    return torch.frexp(x)[1] - 1


def _scaled(x, kind):
    """x [rows, k] float32 -> (elements' values [rows, blocks, 32], scale exponents [rows, blocks, 1]); k is filled up with zeros."""
    rows, k = x.shape
    blocks = -(-k // 32)
    wide = torch.zeros(rows, 32 * blocks, dtype=x.dtype, device=x.device)
    wide[:, :k] = x
    wide = wide.view(rows, blocks, 32)
    part, top = torch.frexp(wide.abs().amax(-1, keepdim=True))
    limit, at = math.frexp(LIMIT[kind])
    e = torch.where(part > 0, top - at + (part > limit), -127).clamp(min=-127)
    s = torch.ldexp(wide, -e)
    low, bits = SMALLEST[kind]
    step = _exponents(s).clamp(min=low) - bits
    s = torch.ldexp(torch.round(torch.ldexp(s, -step)), step)
    return s.clamp(-LARGEST[kind], LARGEST[kind]), e


def _rounded(x, kind):
    """The values that x [rows, k] stands for in the format, float32."""
    s, e = _scaled(x, kind)
    return torch.ldexp(s, e).view(x.shape[0], -1)[:, :x.shape[1]]


def _codes(x):
    """A matrix as a checkpoint holds it: e2m1 codes two to a byte (the first in the low half) [rows, ceil(k / 2)], and scale bytes [rows, ceil(k / 32)]."""
    s, e = _scaled(x, "e2m1")
    magnitudes = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=x.device)
    c = torch.searchsorted(magnitudes, s.abs()) + 8 * (s < 0)
    c = c.view(x.shape[0], -1)
    pairs = (c[:, 0::2] | (c[:, 1::2] << 4))[:, :-(-x.shape[1] // 2)]
    return pairs.to(torch.uint8).contiguous(), (e.view(x.shape[0], -1) + 127).to(torch.uint8)


def _matrix(codes, scales, k):
    """The matrix that codes and scale bytes stand for, float32 [rows, k]."""
    values = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=codes.device)
    rows, blocks = scales.shape
    wide = torch.zeros(rows, 16 * blocks, dtype=torch.uint8, device=codes.device)
    wide[:, :codes.shape[1]] = codes
    w = torch.empty(rows, 16 * blocks, 2, device=codes.device)
    w[..., 0], w[..., 1] = values[(wide & 15).int()], values[(wide >> 4).int()]
    w = torch.ldexp(w.view(rows, blocks, 32), scales.int().view(rows, blocks, 1) - 127)
    return w.view(rows, -1)[:, :k]


# ------------------------------------------------------------------ inputs

def _rows_like(g, rows, k, dtype=torch.float32):
    """Activations: normal, with a few channels that are some thirty times as large as the others, as a decoder's are."""
    x = torch.randn(rows, k, device=DEVICE, generator=g)
    x *= torch.where(torch.rand(k, device=DEVICE, generator=g) < 0.01, 30.0, 1.0)
    return x.to(dtype)


def _weights(g, n, k):
    return (torch.randn(n, k, device=DEVICE, generator=g) * 0.02).bfloat16()


def prepare(case, seed):
    g = torch.Generator(DEVICE).manual_seed(seed)
    do, rows, k, kind = case["do"], case["rows"], case["k"], case["kind"]
    s = {"case": case}
    if do == "quantise":
        dtype = getattr(torch, case["dtype"])
        s["x"] = _weights(g, rows, k).to(dtype) if kind == "e2m1" else _rows_like(g, rows, k, dtype)
    elif do == "norm":
        s["x"] = _rows_like(g, rows, k)
        s["add"] = _rows_like(g, case["shares"] * rows, k).view(case["shares"], rows, k) * 0.3
        s["weight"] = 1.0 + 0.2 * torch.randn(k, device=DEVICE, generator=g)
        s["total"] = torch.empty_like(s["x"])
    else:
        s["x"] = _rows_like(g, rows, k, torch.bfloat16)
        s["matrices"] = [(*_codes(_weights(g, case["n"], k).float()), k) for _ in range(2 if do == "gated" else 1)]
        if do == "product" and case["to"] == "store":
            s["bias"] = torch.randn(case["n"], device=DEVICE, generator=g) * 0.1
        elif do == "product":
            s["stream"] = torch.randn(rows, case["n"], device=DEVICE, generator=g) * 4.0
    if own:      # what an engine keeps: the matrices in the order of the kernels, and room for rows on their way
        from alofa_amd import ops
        s["rows"] = ops.MXRows(rows, k, kind, DEVICE)
        if "matrices" in s:
            s["laid"] = [ops.mx_from_codes(codes, scales, k, "e2m1") for codes, scales, k in s["matrices"]]
        if do == "gated":
            s["act"] = ops.MXRows(rows, case["n"], kind, DEVICE)
    return s


def _run_own(s):
    from alofa_amd import ops
    case = s["case"]
    do, rows, q = case["do"], case["rows"], s["rows"]
    if do == "norm":
        ops.rmsnorm_mx(q, s["x"], s["weight"], EPS, add=s["add"], total=s["total"])
        out = torch.empty(rows, case["k"], dtype=torch.bfloat16, device=DEVICE)
        ops.mx_values(out, q)
        return s["total"], out
    ops.mx_quantize(q, s["x"])
    if do == "quantise":
        out = torch.empty(rows, case["k"], dtype=torch.bfloat16, device=DEVICE)
        ops.mx_values(out, q)
    elif do == "gated":
        ops.gemm_swiglu_mx(s["act"], q, *s["laid"])
        out = torch.empty(rows, case["n"], dtype=torch.bfloat16, device=DEVICE)
        ops.mx_values(out, s["act"])
    elif case["to"] == "store":
        out = torch.empty(rows, case["n"], dtype=torch.bfloat16, device=DEVICE)
        ops.gemm_mx(out, q, s["laid"][0], s["bias"])
    else:
        out = s["stream"]
        ops.gemm_mx(out, q, s["laid"][0], add_to_out=True)
    return out


def run(s):
    if own:
        return _run_own(s)
    case = s["case"]
    do, kind = case["do"], case["kind"]
    if do == "quantise":
        return _rounded(s["x"].float(), kind).bfloat16()
    if do == "norm":
        add = s["add"][0]
        for share in s["add"][1:]:
            add = add + share
        torch.add(s["x"], add, out=s["total"])
        t = s["total"].double()      # (a last bit decides which of two elements a value next to their middle becomes)
        y = t / torch.sqrt(t.square().mean(-1, keepdim=True) + EPS) * s["weight"].double()
        return s["total"], _rounded(y, kind).bfloat16()
    x = _rounded(s["x"].float(), kind)
    products = [x @ _matrix(*m).t() for m in s["matrices"]]
    if do == "gated":
        gate, up = products
        return _rounded(gate / (1.0 + torch.exp(-gate)) * up, kind).bfloat16()
    if case["to"] == "store":
        return (products[0] + s["bias"]).bfloat16()
    return s["stream"].add_(products[0])


def work(case):
    do, rows, k = case["do"], case["rows"], case["k"]
    held = (0.5 if case["kind"] == "e2m1" else 1.0) + 1.0 / 32.0      # bytes of a value of rows, of a matrix (below)
    if do == "quantise":      # numbers in, what is held written and read, values out
        return {"bytes": rows * k * ((2 if case["dtype"] == "bfloat16" else 4) + 2 * held + 2), "flops": 4 * rows * k}
    if do == "norm":      # stream and shares in, stream and rows out, these read again, values out
        return {"bytes": rows * k * (4 + 4 * case["shares"] + 4 + 2 * held + 2) + 4 * k, "flops": (8 + case["shares"]) * rows * k}
    n = case["n"]
    matrix = n * k * (0.5 + 1.0 / 32.0)
    if do == "gated":
        return {"bytes": rows * k * 2 + 2 * matrix + rows * n * (2 * held + 2), "flops": 4 * rows * n * k}
    return {"bytes": rows * k * 2 + matrix + rows * n * (2 if case["to"] == "store" else 8), "flops": 2 * rows * n * k}


# ------------------------------------------------------------------ the definition, in 64 bits

def _nearest(x, kind):
    """The values that x [rows, k] (float64) stands for, by looking each up among the format's magnitudes."""
    low, bits = SMALLEST[kind]
    grid = [0.0] + [m * 2.0 ** (low - bits) for m in range(1, 2 ** bits)]
    e = low
    while grid[-1] < LARGEST[kind]:
        grid += [(1 + m / 2 ** bits) * 2.0 ** e for m in range(2 ** bits)]
        e += 1
    grid = torch.tensor([v for v in grid if v <= LARGEST[kind]], dtype=torch.float64, device=x.device)
    middles = (grid[1:] + grid[:-1]) / 2
    rows, k = x.shape
    out = torch.empty_like(x)
    for at in range(0, rows, 2048):
        part = torch.nn.functional.pad(x[at:at + 2048], (0, -k % 32))
        part = part.view(part.shape[0], -1, 32)
        top = part.abs().amax(-1, keepdim=True).clamp(min=1e-300)
        e = torch.ceil(torch.log2(top / LIMIT[kind]))
        e = torch.where(torch.exp2(e - 1) * LIMIT[kind] >= top, e - 1, e)      # (a logarithm next to a whole number)
        e = torch.where(torch.exp2(e) * LIMIT[kind] < top, e + 1, e).clamp(min=-127)
        size = part.abs() / torch.exp2(e)
        index = torch.searchsorted(middles, size.contiguous())      # middles below
        tie = (index < len(middles)) & (middles[index.clamp(max=len(middles) - 1)] == size) & (index % 2 == 1)
        value = grid[index + tie.long()] * torch.exp2(e) * torch.sign(part)
        out[at:at + 2048] = value.view(part.shape[0], -1)[:, :k]
    return out


def _matrix64(codes, scales, k):
    c = torch.stack((codes & 15, codes >> 4), -1).view(codes.shape[0], -1)[:, :k].long()
    size = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=codes.device)[c & 7]
    return torch.where(c > 7, -size, size) * torch.exp2(scales.double() - 127).repeat_interleave(32, 1)[:, :k]


def exact(case, seed):
    s = prepare(case, seed)
    do, kind = case["do"], case["kind"]
    if do == "quantise":
        return _nearest(s["x"].double(), kind)
    if do == "norm":
        total = s["x"].double() + s["add"].double().sum(0)
        t = (s["x"] + _added(s["add"])).double()      # (what is normed is the stream as it is kept, 32 bits)
        return total, _nearest(t * torch.rsqrt((t * t).mean(-1, keepdim=True) + EPS) * s["weight"].double(), kind)
    x = _nearest(s["x"].double(), kind)
    y = [torch.matmul(x, _matrix64(*m).t().contiguous()) for m in s["matrices"]]
    if do == "gated":
        return _nearest(y[0] * torch.sigmoid(y[0]) * y[1], kind)
    return y[0] + s["bias"].double() if case["to"] == "store" else y[0] + s["stream"].double()


def _added(shares):
    """The shares of a sum, added in 32 bits in their order."""
    total = shares[0].clone()
    for share in shares[1:]:
        total += share
    return total
