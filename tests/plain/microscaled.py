"""Microscaled rows in plain numpy, 64 bits: blocks of 32 along a row, elements of 4 or 8 bits times a power of two per block."""
import numpy as np

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
E4M3 = np.array([m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8)][:127])      # code 127 is NaN
GRID = {"e2m1": E2M1, "e4m3": E4M3}
LIMIT = {"e2m1": 7.0, "e4m3": 464.0}
BITS = {"e2m1": (0, 1), "e4m3": (-6, 3)}      # exponent of the smallest normal element, bits behind the point


def blocks(x):
    """[rows, k] -> [rows, blocks, 32], filled up with zeros."""
    rows, k = x.shape
    wide = np.zeros((rows, -(-k // 32) * 32))
    wide[:, :k] = x
    return wide.reshape(rows, -1, 32)


def scale_exponents(x, kind):
    """e of every block [rows, blocks]; 128 (the byte 255) where a block has an infinity or a NaN."""
    top = np.abs(blocks(np.where(np.isfinite(x), x, 0.0))).max(-1)
    e = np.full(top.shape, -127)
    for at in range(-127, 128):      # the smallest power of two that is large enough
        e = np.where(top > LIMIT[kind] * 2.0 ** at, at + 1, e)
    return np.where(np.isfinite(blocks(x)).all(-1), e, 128)


def codes(x, kind):
    """(element codes [rows, blocks * 32], scale bytes [rows, blocks]) of float64 rows."""
    e = scale_exponents(x, kind)
    with np.errstate(invalid="ignore"):
        size = np.abs(blocks(np.where(np.isfinite(x), x, 0.0))) / np.exp2(np.where(e == 128, 0, e).astype(float))[..., None]
    grid = GRID[kind]
    middles = (grid[1:] + grid[:-1]) / 2
    index = np.searchsorted(middles, size)
    tie = (index < len(middles)) & (middles[np.minimum(index, len(middles) - 1)] == size) & (index % 2 == 1)
    code = index + tie
    sign = len(grid) + len(grid) % 2      # 8, 128
    code = code + sign * np.signbit(blocks(np.where(np.isfinite(x), x, 0.0)))
    return code.reshape(x.shape[0], -1), (e + 127).astype(np.uint8)


def values(code, scales, k, kind):
    """The values behind element codes [rows, blocks * 32] and scale bytes."""
    grid = np.concatenate([E4M3, [np.nan], -E4M3, [np.nan]]) if kind == "e4m3" else np.concatenate([E2M1, -E2M1])
    v = grid[code].reshape(code.shape[0], -1, 32) * np.exp2(scales.astype(float) - 127)[..., None]
    v = np.where((scales == 255)[..., None], np.nan, v)
    return v.reshape(code.shape[0], -1)[:, :k]


def rounded(x, kind):
    """The values that float64 rows stand for in the format."""
    return values(*codes(x, kind), x.shape[1], kind)


def half_step(size, e, kind):
    """Half the distance of elements around magnitudes ``size`` [rows, k] under the scales 2^e [rows, blocks]."""
    low, bits = BITS[kind]
    s = np.exp2(e.astype(float)).repeat(32, axis=1)[:, :size.shape[1]]
    binade = np.floor(np.log2(np.maximum(size / s, 2.0 ** low)))
    return s * np.exp2(binade - bits) / 2


def norm(x, w, eps):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w


def silu(z):
    return z / (1 + np.exp(-z))


def gelu_tanh(z):
    return z / 2 * (1 + np.tanh(np.sqrt(2 / np.pi) * (z + 0.044715 * z ** 3)))


# ------------------------------------------------------------- a decoder whose matrices are e2m1 and whose products read e4m3

MATRICES = ("self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj", "self_attn.o_proj", "mlp.gate_proj", "mlp.up_proj", "mlp.down_proj")


def matrices_rounded(w, cfg):
    """The weights with every layer's seven matrices as e2m1."""
    out = dict(w)
    for i in range(cfg["L"]):
        for name in MATRICES:
            name = f"model.layers.{i}.{name}.weight"
            out[name] = rounded(w[name].astype(np.float64), "e2m1").astype(np.float32)
    return out


def forward_logits(w, cfg, ids, store=lambda x: x):
    """As ``plain.model.forward_logits`` with the matrices of ``matrices_rounded`` and what every product of a layer reads as e4m3. ``store``: applied to queries, keys, values, attention's output and the final norm."""
    from . import model as pm
    T, F32 = len(ids), np.float32
    q8 = lambda x: rounded(x.astype(np.float64), "e4m3").astype(F32)      # noqa: E731
    positions = np.arange(T)
    cos, sin = pm.rope_table(T, cfg["d"], cfg["theta"])
    hidden = pm.embed(w["model.embed_tokens.weight"], ids)
    for i in range(cfg["L"]):
        p = f"model.layers.{i}."
        a = p + "self_attn."
        n = q8(pm.rmsnorm(hidden, w[p + "input_layernorm.weight"], cfg["eps"]))
        q, k, v = (store(pm.linear(n, w[a + c + "_proj.weight"], w[a + c + "_proj.bias"])) for c in "qkv")
        q, k = (store(pm.rope_apply(x, cos, sin, positions, cfg["d"])) for x in (q, k))
        o = q8(store(pm.attention(q, k, v, cfg["H"], cfg["Hkv"], cfg["d"], cfg["windows"][i])))
        hidden = pm.add(hidden, pm.linear(o, w[a + "o_proj.weight"]))
        n = q8(pm.rmsnorm(hidden, w[p + "post_attention_layernorm.weight"], cfg["eps"]))
        act = q8(pm.swiglu(pm.linear(n, w[p + "mlp.gate_proj.weight"]), pm.linear(n, w[p + "mlp.up_proj.weight"])))
        hidden = pm.add(hidden, pm.linear(act, w[p + "mlp.down_proj.weight"]))
    y = store(pm.rmsnorm(hidden, w["model.norm.weight"], cfg["eps"]))
    return pm.linear(y, pm.output_matrix(w, cfg))
