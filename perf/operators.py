"""Cases of the layer norm, dropout and 8-bit product operators.

Each case is one pass as a user's program makes it.  ``own`` chooses between the plain
form (elementary torch operations in 32 bits) and this package's operators.

* ``norm``: layer norm over the last dimension of [rows, c] (``layout`` "rows") or over
  the channels of [n, c, v] ("channels"); with ``train`` also dx, dw and db.
* ``drop``: dropout of ``size`` elements from a counter-based generator, optionally
  added to a residual; with ``train`` also dx.
* ``int8``: 16- or 32-bit activations quantised with one scale for each token, times
  8-bit weights with one scale for each output channel, plus bias.
"""

import math

import numpy as np
import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_TINY = 127.0 * 2.0 ** -126  # the least row maximum that a token's scale is made from
_EPS = 1e-6

# The largest of everything: MedNeXt's outermost level, 32 channels at 128^3 voxels.
_MOST_ELEMENTS = 32 * 128 ** 3
_MOST_MACS = 32768 * 1024 * 4096


def listed():
    return [
        # one token of the widest level at inference: latency alone
        dict(name="norm one token", op="norm", layout="rows", dtype="bf16", n=1, rows=1, c=512, train=False),
        # a token mixer's training step on wide rows
        dict(name="norm rows train", op="norm", layout="rows", dtype="bf16", n=1, rows=16384, c=1024, train=True),
        # the outermost level of a 128^3 patch, trained: the largest
        dict(name="norm level 0 train", op="norm", layout="channels", dtype="bf16", n=1, rows=128 ** 3, c=32, train=True),
        # an odd patch in 32 bits: no row starts on a vector's boundary
        dict(name="norm odd patch train", op="norm", layout="channels", dtype="f32", n=2, rows=33 * 35 * 37, c=96, train=True),
        # inference on a middle level, two patches
        dict(name="norm level 2 forward", op="norm", layout="channels", dtype="f16", n=2, rows=32 ** 3, c=128, train=False),
        # the logits of one deep-supervision head, sampled for uncertainty at inference
        dict(name="drop small head", op="drop", dtype="f32", size=3 * 8 ** 3, p=0.5, residual=False, train=False),
        # the outermost level's residual branch, trained
        dict(name="drop level 0 train", op="drop", dtype="bf16", size=32 * 128 ** 3, p=0.1, residual=True, train=True),
        # an odd patch, no residual
        dict(name="drop odd patch train", op="drop", dtype="f16", size=64 * 33 * 35 * 37 + 5, p=0.2, residual=False, train=True),
        # one token through the widest level's expansion: the weights' bytes count
        dict(name="int8 one token", op="int8", layout="rows", dtype="bf16", n=1, rows=1, k=512, out=2048),
        # the bottleneck's compression, 8^3 voxels
        dict(name="int8 bottleneck", op="int8", layout="channels", dtype="bf16", n=1, rows=512, k=2048, out=512),
        # the outermost level's expansion: activations' bytes count
        dict(name="int8 level 0", op="int8", layout="channels", dtype="bf16", n=1, rows=128 ** 3, k=32, out=64),
        # wide rows: the tensor cores count
        dict(name="int8 wide rows", op="int8", layout="rows", dtype="bf16", n=1, rows=32768, k=1024, out=4096),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("norm", "drop", "int8"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    most = _MOST_ELEMENTS // (2 if dtype == "f32" else 1)
    if op == "drop":
        size = _spread(rng, 1000, most)
        size = size // 1024 * 1024 if size > 4096 and rng.random() < 0.5 else size  # whole volumes are as usual as odd ones
        return dict(op=op, dtype=dtype, size=size, p=round(rng.uniform(0.02, 0.6), 3), residual=rng.random() < 0.5,
                    train=rng.random() < 0.5)
    layout = rng.choice(("rows", "channels"))
    n = rng.choice((1, 1, 2, 3)) if layout == "channels" else 1
    if op == "norm":
        c = _spread(rng, 16, 4096 if layout == "rows" else 1024)
        c = c // 16 * 16 if rng.random() < 0.6 else c  # model widths, and odd ones
        rows = _spread(rng, 1, most // (c * n))
        rows = rows // 8 * 8 if rows > 64 and rng.random() < 0.6 else rows
        return dict(op=op, layout=layout, dtype=dtype, n=n, rows=rows, c=c, train=rng.random() < 0.6)
    k, out = _spread(rng, 32, 4096), _spread(rng, 32, 4096)
    if rng.random() < 0.7:
        k, out = k // 32 * 32, out // 32 * 32
    rows = _spread(rng, 1, max(2, min(128 ** 3, most // (n * max(k, out)), _MOST_MACS // (n * k * out))))
    rows = rows // 8 * 8 if rows > 64 and rng.random() < 0.6 else rows
    return dict(op=op, layout=layout, dtype=dtype, n=n, rows=rows, k=k, out=out)


def _shape(case, width):
    return (case["rows"], width) if case["layout"] == "rows" else (case["n"], width, case["rows"])


def _wide(case, v):
    """A vector over the channels, shaped to meet the case's tensors."""
    return v if case["layout"] == "rows" else v[:, None]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    state = {"case": case}
    if case["op"] == "norm":
        c = case["c"]
        # channels with means and spreads of their own, as a network's features have
        x = normal(*_shape(case, c)) * _wide(case, normal(c).abs() + 0.3) + _wide(case, 0.5 * normal(c))
        state.update(x=x.to(dtype), weight=1.0 + 0.2 * normal(c), bias=0.1 * normal(c))
        if case["train"]:
            state["dy"] = normal(*_shape(case, c)).to(dtype)
            for name in ("x", "weight", "bias"):
                state[name].requires_grad_(True)
    elif case["op"] == "drop":
        # seed and offset of the generator, on the GPU as a captured training step keeps them
        state["rng"] = torch.tensor([int(seed) * 1000003 + 12345, int(seed) % 977], device="cuda")
        state["x"] = normal(case["size"]).to(dtype)
        if case["residual"]:
            state["residual"] = normal(case["size"]).to(dtype)
        if case["train"]:
            state["dy"] = normal(case["size"]).to(dtype)
            state["x"].requires_grad_(True)
    else:
        k, out = case["k"], case["out"]
        # a few channels are much larger than the rest, as activations have them
        spread = torch.where(torch.rand(k, generator=gen, device="cuda") < 0.02, 8.0, 1.0)
        state["x"] = (normal(*_shape(case, k)) * _wide(case, spread)).to(dtype)
        # 8-bit weights as a program keeps them: rows padded to 16 bytes
        held = torch.zeros((out, (k + 15) // 16 * 16), dtype=torch.int8, device="cuda")
        held[:, :k] = (normal(out, k) * 40).round().clamp(-127, 127).to(torch.int8)
        state["weight"] = held[:, :k]
        state["scale"] = (0.5 + torch.rand(out, generator=gen, device="cuda")) / (40 * math.sqrt(k))
        state["bias"] = 0.1 * normal(out)
    return state


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    import mednext_accel_b200 as mx

    case = state["case"]
    if case["op"] == "drop":
        y = mx.dropout(state["x"], case["p"], state["rng"], residual=state.get("residual"))
        if case["train"]:
            return {"y": y, "dx": torch.autograd.grad(y, state["x"], state["dy"])[0]}
        return {"y": y}
    dim = -1 if case["layout"] == "rows" else 1
    if case["op"] == "norm":
        x, weight, bias = state["x"], state["weight"], state["bias"]
        y = mx.layer_norm(x, weight, bias, eps=_EPS, dim=dim)
        if case["train"]:
            dx, dw, db = torch.autograd.grad(y, (x, weight, bias), state["dy"])
            return {"y": y, "dx": dx, "dw": dw, "db": db}
        return {"y": y}
    return {"y": mx.int8_linear(state["x"], state["weight"], state["scale"], state["bias"], dim=dim)}


# --------------------------------------------------------------------------- plain forms
def _run_plain(state):
    with torch.no_grad():
        return {"norm": _plain_norm, "drop": _plain_drop, "int8": _plain_int8}[state["case"]["op"]](state)


def _plain_norm(state):
    case, dtype = state["case"], state["x"].dtype
    dim = -1 if case["layout"] == "rows" else 1
    tokens = [0] if dim == -1 else [0, 2]
    x, w = state["x"].float(), _wide(case, state["weight"])
    d = x - x.mean(dim, keepdim=True)
    r = ((d * d).mean(dim, keepdim=True) + _EPS).rsqrt()
    xh = d * r
    y = (xh * w + _wide(case, state["bias"])).to(dtype)
    if not case["train"]:
        return {"y": y}
    dy = state["dy"].float()
    g = dy * w
    dx = r * (g - g.mean(dim, keepdim=True) - xh * (g * xh).mean(dim, keepdim=True))
    return {"y": y, "dx": dx.to(dtype), "dw": (dy * xh).sum(tokens), "db": dy.sum(tokens)}


def _philox(seed, offset, count):
    """Philox4x32-10: [count, 4] words of 32 bits, held in 64; counter (i, offset), key seed."""
    mask = 0xFFFFFFFF
    i = torch.arange(count, device=seed.device)
    a, b = i & mask, (i >> 32) & mask
    c, d = (offset & mask).expand(count), ((offset >> 32) & mask).expand(count)
    k0, k1 = seed & mask, (seed >> 32) & mask
    for _ in range(10):
        p, q = a * 0xD2511F53, c * 0xCD9E8D57  # modulo 2^64: the bits are those of the unsigned product
        a, b, c, d = ((q >> 32) & mask) ^ b ^ k0, q & mask, ((p >> 32) & mask) ^ d ^ k1, p & mask
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    return torch.stack((a, b, c, d), 1)


def _plain_drop(state):
    case, x = state["case"], state["x"]
    size, t = case["size"], round(case["p"] * 65536)
    words = _philox(state["rng"][0], state["rng"][1], (size + 7) // 8)
    words = torch.stack((words & 0xFFFF, words >> 16), 2).reshape(-1)[:size]
    keep = words >= t
    scale = 65536.0 / (65536 - t)
    y = torch.where(keep, x.float() * scale, 0.0)
    if case["residual"]:
        y = y + state["residual"].float()
    if not case["train"]:
        return {"y": y.to(x.dtype)}
    return {"y": y.to(x.dtype), "dx": torch.where(keep, state["dy"].float() * scale, 0.0).to(x.dtype)}


def _plain_int8(state):
    case, x = state["case"], state["x"].float()
    dim = -1 if case["layout"] == "rows" else 1
    most = x.abs().amax(dim, keepdim=True).clamp_min(_TINY)
    q = (x * torch.div(torch.full_like(most, 127.0), most)).round()  # a number over a tensor would be its reciprocal, rounded twice
    w = state["weight"].float()
    acc = q @ w.t() if dim == -1 else w @ q
    y = acc * torch.div(most, torch.full_like(most, 127.0)) * _wide(case, state["scale"]) + _wide(case, state["bias"])
    return {"y": y.to(state["x"].dtype)}


# --------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "drop": _exact_drop, "int8": _exact_int8}[case["op"]](case, state)


def _tokens(case, t):
    """[tokens, width] in 64 bits from either layout."""
    t = t.double()
    return t if case["layout"] == "rows" else t.transpose(1, 2).reshape(-1, t.shape[1])


def _laid_out(case, t):
    """The case's layout from [tokens, width]."""
    if case["layout"] == "rows":
        return t
    return t.reshape(case["n"], case["rows"], -1).transpose(1, 2).contiguous()


def _exact_norm(case, state):
    x = _tokens(case, state["x"])
    w, b = state["weight"].double(), state["bias"].double()
    var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
    sd = torch.sqrt(var + _EPS)
    out = {"y": _laid_out(case, torch.addcmul(b, (x - mean) / sd, w))}
    if case["train"]:
        dy = _tokens(case, state["dy"])
        c = x.shape[1]
        # the Jacobian of (x - mean) / sd applied to dy w, term by term
        g, d = dy * w, x - mean
        dx = g / sd - g.sum(1, keepdim=True) / (c * sd) - d * (g * d).sum(1, keepdim=True) / (c * sd ** 3)
        out.update(dx=_laid_out(case, dx), dw=torch.einsum("tc,tc->c", dy, d / sd), db=torch.einsum("tc->c", dy))
    return out


def _exact_drop(case, state):
    seed, offset = (int(v) % 2 ** 64 for v in state["rng"].tolist())
    size, low = case["size"], np.uint64(0xFFFFFFFF)
    word = [np.uint32(v & 0xFFFFFFFF) for v in (seed, seed >> 32, offset, offset >> 32)]
    kept = np.empty((size + 7) // 8 * 8, dtype=bool)
    t = round(case["p"] * 65536)
    for begin in range(0, len(kept) // 8, 1 << 20):
        i = np.arange(begin, min(begin + (1 << 20), len(kept) // 8), dtype=np.uint64)
        ctr = [(i & low).astype(np.uint32), (i >> np.uint64(32)).astype(np.uint32),
               np.full(len(i), word[2]), np.full(len(i), word[3])]
        for turn in range(10):
            key = [np.uint32((int(word[0]) + turn * 0x9E3779B9) % 2 ** 32), np.uint32((int(word[1]) + turn * 0xBB67AE85) % 2 ** 32)]
            first = ctr[0].astype(np.uint64) * np.uint64(0xD2511F53)
            second = ctr[2].astype(np.uint64) * np.uint64(0xCD9E8D57)
            ctr = [(second >> np.uint64(32)).astype(np.uint32) ^ ctr[1] ^ key[0], second.astype(np.uint32),
                   (first >> np.uint64(32)).astype(np.uint32) ^ ctr[3] ^ key[1], first.astype(np.uint32)]
        halves = np.stack(ctr, 1).astype("<u4").view("<u2").reshape(-1)
        kept[8 * begin:8 * begin + len(halves)] = halves >= t
    keep = torch.from_numpy(kept[:size]).cuda()
    scale = 65536.0 / (65536 - t)

    def dropped(v):
        return v.double().mul(scale).masked_fill(~keep, 0.0)

    y = dropped(state["x"])
    out = {"y": y + state["residual"].double() if case["residual"] else y}
    if case["train"]:
        out["dx"] = dropped(state["dy"])
    return out


def _exact_int8(case, state):
    x = _tokens(case, state["x"])
    held = torch.clamp_min(torch.linalg.vector_norm(x, ord=math.inf, dim=1, keepdim=True), _TINY)
    step = held / 127.0
    whole = torch.round(x / step)
    y = torch.addmm(state["bias"].double(), whole * step, (state["weight"].double() * state["scale"].double()[:, None]).t())
    return {"y": _laid_out(case, y)}


# --------------------------------------------------------------------------- floors
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "drop":
        n, train = case["size"], case["train"]
        return {"bytes": n * size * (2 + int(case["residual"]) + 2 * int(train)), "flops": n * 2 * (1 + int(train))}
    tokens = case["n"] * case["rows"]
    if case["op"] == "norm":
        n, c, train = tokens * case["c"], case["c"], case["train"]
        return {"bytes": n * size * (4 if train else 2) + 4 * c * (4 if train else 2), "flops": n * (22 if train else 8)}
    k, out = case["k"], case["out"]
    return {"bytes": tokens * (k + out) * size + out * k + 8 * out, "flops": 2 * tokens * k * out}
