"""Layer norm, dropout and the residual add that joins them: the cases their time is measured on.

Three operators of `segmentation_amd.ops`, each in its forward form and in the form a training step needs:

* layer norm over the channels of a row (`layer_norm_fwd`, `layer_norm_backward`);
* dropout whose mask comes from a counter-based generator and is never stored (`dropout`, used again on the gradient);
* h = residual + dropout(x), y = layer_norm(h) in one pass each way (`dropout_add_layer_norm_fwd`, `_backward`).

A case is one pass: "eval" (the forward) or "train" (forward and all gradients).  Rows are voxels, points or tokens;
`pad` further columns lie behind every row of the inputs, as behind a slice of concatenated features.
"""
import functools

import torch

#: False: the operators in elementary torch operations.  True: the framework's kernels.
own = False

EPS = 1e-5

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def _case(name, op, mode, rows, cols, x, w, stream=None, p=0.0, pad=0):
    """x: type of the activations, w: of weight and bias, stream: of the residual stream (add), p: dropout."""
    return {"name": name, "op": op, "mode": mode, "rows": rows, "cols": cols, "x": x, "w": w, "stream": stream or x,
            "p": p, "pad": pad}


def listed():
    return [
        # one feature row through an inference head: nothing but latency
        _case("ln_one_row", "ln", "eval", 1, 768, "bf16", "f32"),
        # finest level of the benchmark scene at the width of the last decoder block
        _case("ln_level0_train", "ln", "train", 273080, 96, "f32", "f32"),
        # 768-channel features of the second level, mixed precision
        _case("ln_features_train", "ln", "train", 75401, 768, "bf16", "f32"),
        # odd channel count, rows sliced out of a wider tensor
        _case("ln_ragged_train", "ln", "train", 3493, 1001, "f16", "f16", pad=7),
        # a wide layer over a long batch, inference
        _case("ln_wide", "ln", "eval", 8192, 8192, "bf16", "bf16"),
        # coarsest level of the scene, training
        _case("dropout_level4_train", "dropout", "train", 739, 256, "f32", "f32", p=0.1),
        # finest level of the scene, training
        _case("dropout_level0_train", "dropout", "train", 273080, 96, "f32", "f32", p=0.1),
        # a wide activation in mixed precision
        _case("dropout_wide_train", "dropout", "train", 16384, 4096, "bf16", "bf16", p=0.2),
        # a few tokens through the residual stream of a wide model, inference: no dropout
        _case("add_tokens", "add", "eval", 8, 4096, "bf16", "bf16"),
        # second level of the scene, training
        _case("add_level1_train", "add", "train", 75401, 256, "f32", "f32", p=0.1),
        # bf16 branch on a residual stream held in 32 bits
        _case("add_stream_train", "add", "train", 30001, 768, "bf16", "f32", stream="f32", p=0.1),
        # a wide model's block, everything in bf16: the largest case
        _case("add_wide_train", "add", "train", 16384, 4096, "bf16", "bf16", p=0.1),
    ]


def draw(rng):
    op = rng.choice(["ln", "dropout", "add", "add"])
    x = rng.choice(["f32", "bf16", "f16"])
    mode = rng.choice(["eval", "train", "train"])
    cols = int(16 * 512 ** rng.random())
    cols = min(8192, cols if rng.random() < 0.4 else -(-cols // 16) * 16)
    most = (1 << 24) // cols  # values of one tensor: a quarter of the largest listed case
    rows = max(1, min(300000, int(most ** rng.random()), most))
    p = rng.choice([0.05, 0.1, 0.25, 0.5]) if op == "dropout" else rng.choice([0.0, 0.1, 0.3]) if op == "add" else 0.0
    stream = rng.choice([x, "f32"]) if op == "add" else x
    # x / (1 - p) lies on the borders of a 16-bit stream's rounding often enough for 32 and 64 bits to part there by 1e-4
    # of the weight's gradient, which a gradient in 32 bits would show
    w = x if op == "add" and stream != "f32" and p > 0 else rng.choice([x, "f32"])
    return {"op": op, "mode": mode, "rows": rows, "cols": cols, "x": x, "w": w, "stream": stream, "p": p,
            "pad": rng.choice([0, 0, 0, 5, 64])}


def _randn(g, rows, cols, pad, dtype, scale=1.0, shift=0.0):
    t = torch.empty((rows, cols + pad), dtype=torch.float32, device="cuda").normal_(generator=g)
    return t.mul_(scale).add_(shift).to(dtype)[:, :cols]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, cols, pad = case["rows"], case["cols"], case["pad"]
    x, w, stream = _TYPES[case["x"]], _TYPES[case["w"]], _TYPES[case["stream"]]
    s = {"op": case["op"], "mode": case["mode"], "p": case["p"], "seed": 0x5EED0000 + seed, "offset": 11 + seed,
         "x": _randn(g, rows, cols, pad, x, 1.5, 0.25)}
    if case["op"] != "dropout":
        s["weight"] = _randn(g, 1, cols, 0, w, 0.2, 1.0).reshape(-1)
        s["bias"] = _randn(g, 1, cols, 0, w, 0.3).reshape(-1)
    if case["op"] == "add":
        s["residual"] = _randn(g, rows, cols, pad, stream, 2.0)
    if case["mode"] == "train":
        s["dy"] = _randn(g, rows, cols, pad, x)
        if case["op"] == "add":
            s["dh"] = _randn(g, rows, cols, pad, stream)
    return s


def work(case):
    n, c, train = case["rows"] * case["cols"], case["cols"], case["mode"] == "train"
    x, w, h = _BYTES[case["x"]], _BYTES[case["w"]], _BYTES[case["stream"]]
    if case["op"] == "dropout":
        # forward: x -> y; backward: dy -> dx.  Flops: the products, not the generator's integer work.
        return {"bytes": n * 2 * x * (2 if train else 1), "flops": n * (2 if train else 1)}
    wide = 2 * c * w
    if case["op"] == "ln":
        # forward: x, weight, bias -> y; backward: x again, dy -> dx, dweight, dbias
        return {"bytes": n * 2 * x + wide + (n * 3 * x + c * w + wide if train else 0), "flops": n * (8 + (14 if train else 0))}
    # forward: x, residual -> h, y; backward: h, dy, dh -> dx, dresidual, dweight, dbias
    back = n * (h + x + h + h + x) + c * w + wide
    return {"bytes": n * (2 * x + 2 * h) + wide + (back if train else 0), "flops": n * (10 + (17 if train else 0))}


# ---------------------------------------------------------------- plain forms
def _round(c, r, seed):
    """One round of Philox 4x32 (Salmon et al., SC 2011): c = four words in int64 tensors."""
    m = 0xFFFFFFFF
    k0, k1 = ((seed & m) + r * 0x9E3779B9) & m, ((seed >> 32 & m) + r * 0xBB67AE85) & m
    a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
    return [(b >> 32 & m) ^ c[1] ^ k0, b & m, (a >> 32 & m) ^ c[3] ^ k1, a & m]


def _keep(rows, cols, p, seed, offset, device):
    """Where (row, column) is kept: word column % 4 of block (column / 4, row, offset) is at least p * 2^32; 7 rounds."""
    chunk = torch.arange((cols + 3) // 4, device=device)[None, :].expand(rows, -1)
    row = torch.arange(rows, device=device)[:, None].expand(-1, chunk.shape[1])
    word = torch.full((1, 1), offset & 0xFFFFFFFF, device=device), torch.full((1, 1), offset >> 32, device=device)
    c = functools.reduce(lambda c, r: _round(c, r, seed), range(7), [chunk, row, *word])
    return torch.stack(torch.broadcast_tensors(*c), -1).reshape(rows, -1)[:, :cols] >= round(p * 2 ** 32)


def _drop(x, keep, p):
    return x if keep is None else torch.where(keep, x * (1.0 / (1.0 - p)), 0.0)


def _norm(x, weight, bias):
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = 1.0 / torch.sqrt((d * d).mean(1, keepdim=True) + EPS)
    return d * rstd * weight.float() + bias.float(), mean, rstd


def _norm_grad(x, dy, mean, rstd, weight):
    hat, gw = (x - mean) * rstd, dy * weight.float()
    dx = (gw - gw.mean(1, keepdim=True) - hat * (gw * hat).mean(1, keepdim=True)) * rstd
    return dx, (dy * hat).sum(0), dy.sum(0)


def _plain(s):
    x, p, train = s["x"], s["p"], s["mode"] == "train"
    keep = _keep(x.shape[0], x.shape[1], p, s["seed"], s["offset"], x.device) if p > 0 else None
    if s["op"] == "dropout":
        out = {"y": _drop(x.float(), keep, p).to(x.dtype)}
        if train:
            # the mask is not kept between the passes
            keep = _keep(x.shape[0], x.shape[1], p, s["seed"], s["offset"], x.device)
            out["dx"] = _drop(s["dy"].float(), keep, p).to(x.dtype)
        return out
    weight, bias, h = s["weight"], s["bias"], x
    out = {}
    if s["op"] == "add":
        # the stream is held in its own type, and the norm reads what is held
        out["h"] = h = (s["residual"].float() + _drop(x.float(), keep, p)).to(s["residual"].dtype)
    y, mean, rstd = _norm(h.float(), weight, bias)
    out["y"] = y.to(x.dtype)  # the row statistics stay between the passes
    if train:
        dx, dweight, dbias = _norm_grad(h.float(), s["dy"].float(), mean, rstd, weight)
        if s["op"] == "add":
            dx = dx + s["dh"].float()
            out["dresidual"] = dx.to(h.dtype)
            keep = _keep(x.shape[0], x.shape[1], p, s["seed"], s["offset"], x.device) if p > 0 else None
            dx = _drop(dx, keep, p)
        out |= {"dx": dx.to(x.dtype), "dweight": dweight.to(weight.dtype), "dbias": dbias.to(bias.dtype)}
    return out


# ---------------------------------------------------------------- the framework's calls
def _own(s):
    from segmentation_amd import ops
    x, p, train = s["x"], s["p"], s["mode"] == "train"
    rng = {"p": p, "seed": s["seed"], "offset": s["offset"]}
    if s["op"] == "dropout":
        out = {"y": ops.dropout(x, **rng)}
        if train:
            out["dx"] = ops.dropout(s["dy"], **rng)
        return out
    weight, bias = s["weight"], s["bias"]
    if s["op"] == "ln":
        y, mean, rstd = ops.layer_norm_fwd(x, weight, bias, EPS)
        out = {"y": y}
        if train:
            out["dx"], out["dweight"], out["dbias"] = ops.layer_norm_backward(x, s["dy"], mean, rstd, weight)
        return out
    y, h, mean, rstd = ops.dropout_add_layer_norm_fwd(x, s["residual"], weight, bias, EPS, **rng)
    out = {"h": h, "y": y}
    if train:
        out["dx"], out["dresidual"], out["dweight"], out["dbias"] = ops.dropout_add_layer_norm_backward(
            h, s["dy"], s["dh"], mean, rstd, weight, **rng)
    return out


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------- in 64 bits, from the definitions
def _high_low(a, b):
    """High and low word of the 64-bit product of 32-bit words a (tensor) and b, by 16-bit limbs."""
    ah, al, bh, bl = a // 65536, a % 65536, b // 65536, b % 65536
    mid = ah * bl + (al * bl) // 65536
    low = mid % 65536 + al * bh
    return ah * bh + mid // 65536 + low // 65536, (low % 65536) * 65536 + (al * bl) % 65536


def _factor64(case, seed, device):
    """1 / (1 - p) where a value is kept, 0 where it is dropped."""
    p, rows, cols = case["p"], case["rows"], case["cols"]
    if p == 0:
        return 1.0
    key, offset = 0x5EED0000 + seed, 11 + seed
    k = [key % 2 ** 32, key // 2 ** 32]
    quad = -(-cols // 4)
    at = torch.arange(rows * quad, device=device)
    w0, w1 = at % quad, at // quad
    w2, w3 = torch.full_like(at, offset % 2 ** 32), torch.full_like(at, offset // 2 ** 32)
    for _ in range(7):
        h0, l0 = _high_low(w0, 0xD2511F53)
        h2, l2 = _high_low(w2, 0xCD9E8D57)
        w0, w1, w2, w3 = torch.bitwise_xor(torch.bitwise_xor(h2, w1), k[0]), l2, torch.bitwise_xor(torch.bitwise_xor(h0, w3), k[1]), l0
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    u = torch.empty((rows, quad * 4), dtype=torch.float64, device=device)
    for j, word in enumerate((w0, w1, w2, w3)):
        u[:, j::4] = word.reshape(rows, quad) / 2.0 ** 32
    return (u[:, :cols] >= round(p * 2 ** 32) / 2.0 ** 32).double() / (1.0 - p)


def exact(case, seed):
    s = prepare(case, seed)
    f = _factor64(case, seed, s["x"].device)
    x, train = s["x"].double(), case["mode"] == "train"
    if case["op"] == "dropout":
        return {"y": x * f, **({"dx": s["dy"].double() * f} if train else {})}
    out, h = {}, x
    if case["op"] == "add":
        out["h"] = s["residual"].double() + x * f
        h = out["h"].to(s["residual"].dtype).double()
    n = case["cols"]
    weight = s["weight"].double()
    mean = h.sum(1) / n
    centred = h - mean[:, None]
    rstd = (centred.square().sum(1) / n + EPS).rsqrt()
    hat = centred.mul_(rstd[:, None])
    out["y"] = torch.addcmul(s["bias"].double(), hat, weight)
    if train:
        dy = s["dy"].double()
        out["dweight"], out["dbias"] = torch.mul(dy, hat).sum(0), dy.sum(0)
        g = dy * weight
        dot = torch.mul(g, hat).sum(1) / n
        dh = (g - (g.sum(1) / n)[:, None] - hat * dot[:, None]) * rstd[:, None]
        if case["op"] == "add":
            dh += s["dh"].double()
            out["dresidual"] = dh
            dh = dh * f
        out["dx"] = dh
    return out
