"""CPU restatement of layer norm, dropout and the residual add that joins them, in float64.  Test infrastructure only.

The reference calls nn.LayerNorm and nn.Dropout (mosaic3d/src/models/networks/opensegment3d); the dropout masks here
follow the generator's published definition (Philox 4x32, Salmon et al., SC 2011), written with numpy's 64-bit words."""
import numpy as np
import torch


def philox4x32(counter, key, rounds):
    """counter: four uint32 arrays (broadcast), key: two ints -> four uint32 arrays."""
    mask = np.uint64(0xFFFFFFFF)
    c = [np.asarray(w, dtype=np.uint64) for w in np.broadcast_arrays(*counter)]
    k = [int(key[0]), int(key[1])]
    for _ in range(rounds):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        hi_a, lo_a, hi_b, lo_b = a >> np.uint64(32), a & mask, b >> np.uint64(32), b & mask
        c = [hi_b ^ c[1] ^ np.uint64(k[0]), lo_b, hi_a ^ c[3] ^ np.uint64(k[1]), lo_a]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return [w.astype(np.uint32) for w in c]


def dropout_keep(n, c, p, seed, offset):
    """Bool [n, c]: which values dropout keeps."""
    quads = -(-c // 4)
    words = philox4x32((np.arange(quads)[None, :], np.arange(n)[:, None], offset & 0xFFFFFFFF, offset >> 32),
                       (seed & 0xFFFFFFFF, seed >> 32), 7)
    u = np.stack(words, -1).reshape(n, 4 * quads)[:, :c].astype(np.uint64)
    return torch.from_numpy(u >= np.uint64(round(p * 2 ** 32)))


def dropout(x, p, seed, offset):
    """x [n, c] float64."""
    keep = dropout_keep(x.shape[0], x.shape[1], p, seed, offset)
    return torch.where(keep, x / (1.0 - p) if p < 1.0 else torch.zeros_like(x), torch.zeros_like(x))


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """x [n, c] float64 -> (y, mean [n], rstd [n])."""
    mean = x.mean(1)
    d = x - mean[:, None]
    rstd = 1.0 / torch.sqrt((d * d).mean(1) + eps)
    y = d * rstd[:, None]
    if weight is not None:
        y = y * weight
    if bias is not None:
        y = y + bias
    return y, mean, rstd


def layer_norm_backward(x, dy, mean, rstd, weight=None):
    """(dx, dweight, dbias), everything float64."""
    hat = (x - mean[:, None]) * rstd[:, None]
    g = dy if weight is None else dy * weight
    dx = rstd[:, None] * (g - g.mean(1, keepdim=True) - hat * (g * hat).mean(1, keepdim=True))
    return dx, (dy * hat).sum(0), dy.sum(0)
