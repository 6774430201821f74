"""Layer norm, dropout and their residual add without a GPU: the oracle's generator against its authors' published
known answers, the statistics of a mask, refusals of the tensor-level operators and of the C entry points, modules."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import layer_norm as O
from segmentation_amd import _lib, layers, ops, spunet


@pytest.mark.parametrize("rounds,ctr,key,words", [
    (7, (0, 0, 0, 0), (0, 0), (0x5f6fb709, 0x0d893f64, 0x4f121f81, 0x4f730a48)),
    (10, (0, 0, 0, 0), (0, 0), (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
    (10, (0xffffffff,) * 4, (0xffffffff,) * 2, (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
])
def test_generator_known_answers(rounds, ctr, key, words):
    got = O.philox4x32([np.array([v], dtype=np.uint64) for v in ctr], key, rounds)
    assert tuple(int(w[0]) for w in got) == words


def test_mask_statistics():
    n, c, p = 2000, 500, 0.3
    a, b = O.dropout_keep(n, c, p, 7, 0), O.dropout_keep(n, c, p, 7, 1)
    # means and the agreement of two offsets within 5 standard deviations of independent draws
    sd = (p * (1 - p) / (n * c)) ** 0.5
    assert abs(a.double().mean().item() - (1 - p)) < 5 * sd
    same = (1 - p) ** 2 + p ** 2
    assert abs((a == b).double().mean().item() - same) < 5 * (same * (1 - same) / (n * c)) ** 0.5
    assert abs((a[1:] == a[:-1]).double().mean().item() - same) < 5 * (same * (1 - same) / (n * c)) ** 0.5
    assert O.dropout_keep(3, 5, 0.0, 1, 2).all() and not O.dropout_keep(3, 5, 1.0, 1, 2).any()


def test_refusals_of_the_operators():
    x = torch.zeros(4, 8)
    w = torch.ones(8)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.layer_norm_fwd(x, w, w)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.dropout(x, 0.5)
    with pytest.raises(RuntimeError, match="no CPU path"):
        layers.DropoutAddLayerNorm(8, 0.1)(x, x)
    with pytest.raises(TypeError, match="not supported"):
        ops.layer_norm_fwd(x.double())
    with pytest.raises(TypeError, match="not supported"):
        ops.dropout(x.long(), 0.5)
    with pytest.raises(ValueError, match="weight has shape"):
        ops.layer_norm_fwd(x, torch.ones(7))
    with pytest.raises(TypeError, match="both"):
        ops.layer_norm_fwd(x, w, w.bfloat16())
    with pytest.raises(TypeError, match="both"):
        ops.layer_norm_fwd(x.half(), w.bfloat16())
    with pytest.raises(ValueError, match="1 <= c <="):
        ops.layer_norm_fwd(torch.zeros(2, 16385))
    with pytest.raises(ValueError, match="1 <= c <="):
        ops.layer_norm_fwd(torch.zeros(2, 0))
    with pytest.raises(ValueError, match="1 <= c <="):
        ops.layer_norm_fwd(torch.zeros(()))
    with pytest.raises(ValueError, match="eps"):
        ops.layer_norm_fwd(x, eps=-1e-3)
    with pytest.raises(ValueError, match="eps"):
        ops.layer_norm_fwd(x, eps=float("nan"))
    m = torch.zeros(4)
    with pytest.raises(ValueError, match="dy has shape"):
        ops.layer_norm_backward(x, torch.zeros(4, 7), m, m)
    with pytest.raises(TypeError, match="dy is"):
        ops.layer_norm_backward(x, x.half(), m, m)
    with pytest.raises(ValueError, match="mean has shape"):
        ops.layer_norm_backward(x, x, torch.zeros(3), m)
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError, match="not in"):
            ops.dropout(x, p)
        with pytest.raises(ValueError, match="not in"):
            layers.Dropout(p)
        with pytest.raises(ValueError, match="not in"):
            layers.dropout(x, p)
    with pytest.raises(ValueError, match="64-bit"):
        ops.dropout(x, 0.5, seed=-1)
    with pytest.raises(ValueError, match="64-bit"):
        ops.dropout(x, 0.5, offset=2 ** 64)
    with pytest.raises(ValueError, match="not both"):
        ops.dropout(x, 0.5, seed=1, state=ops.dropout_state(1, "cpu"))
    with pytest.raises(TypeError, match="generator state"):
        ops.dropout(x, 0.5, state=torch.zeros(2))
    with pytest.raises(TypeError, match="generator state"):
        ops.dropout_next(None)
    with pytest.raises(ValueError, match="0..2"):
        ops.dropout_state(-1, "cpu")
    with pytest.raises(ValueError, match="residual has shape"):
        ops.dropout_add_layer_norm_fwd(x, torch.zeros(4, 9))
    with pytest.raises(TypeError, match="the residual is"):
        ops.dropout_add_layer_norm_fwd(x, x.half())
    with pytest.raises(TypeError, match="h is"):
        ops.dropout_add_layer_norm_backward(x.half(), x, None, m, m)
    with pytest.raises(TypeError, match="dh is"):
        ops.dropout_add_layer_norm_backward(x, x, x.half(), m, m)


def test_refusals_of_the_entry_points():
    lib = _lib.load()
    one, odd, null = ctypes.c_void_p(16), ctypes.c_void_p(17), ctypes.c_void_p(0)   # never dereferenced

    def fwd(x=one, ld=8, typ=0, n=4, c=8, w=null, wt=0, eps=1e-5, y=one):
        return lib.m3d_layer_norm_fwd(x, ld, typ, n, c, w, null, wt, eps, y, one, one, null)

    for bad in (dict(typ=3), dict(wt=2), dict(c=0), dict(c=16385), dict(n=-1), dict(n=1 << 32), dict(x=null), dict(y=null),
                dict(x=odd), dict(w=odd), dict(ld=7), dict(ld=(1 << 20) + 1), dict(eps=-1.0), dict(eps=float("nan"))):
        assert fwd(**bad) == -1 and lib.m3d_last_error(), bad
    assert fwd(n=0) == 0

    def bwd(ld=8, ldg=8, n=4, dx=one, ws=one, nb=1 << 20, dw=one):
        return lib.m3d_layer_norm_backward(one, ld, one, ldg, 0, n, 8, one, one, null, 0, dx, dw, null, ws, nb, null)

    assert bwd(ld=7) == -1 and bwd(ldg=7) == -1 and bwd(dx=null) == -1 and bwd(ws=ctypes.c_void_p(20)) == -1
    assert bwd(ws=null) == -2 and bwd(nb=8) == -2 and b"workspace" in lib.m3d_last_error()
    assert bwd(n=0, dw=null) == 0

    def drop(x=one, typ=0, n=4, c=8, p=0.5, ld=8, state=null):
        return lib.m3d_dropout(x, ld, typ, n, c, p, 1, 2, state, one, null)

    for bad in (dict(x=null), dict(x=odd), dict(typ=-1), dict(n=1 << 32), dict(c=0), dict(p=-0.5), dict(p=1.5),
                dict(p=float("nan")), dict(ld=3), dict(state=ctypes.c_void_p(20))):
        assert drop(**bad) == -1, bad
    assert drop(n=0) == 0
    assert lib.m3d_dropout_next(null, 1, one, null) == -1 and lib.m3d_dropout_next(one, 1, odd, null) == -1

    def add(typ=1, stream=0, ldr=8, p=0.1, res=one):
        return lib.m3d_dropout_add_layer_norm_fwd(one, 8, typ, res, ldr, stream, 4, 8, null, null, 0, 1e-5, p, 1, 2, null,
                                                  one, one, one, one, null)

    for bad in (dict(stream=2), dict(typ=0, stream=1), dict(ldr=7), dict(p=2.0), dict(res=null),
                dict(res=ctypes.c_void_p(18))):
        assert add(**bad) == -1, bad

    def addb(dx=one, dr=one, lddh=8, dh=one):
        return lib.m3d_dropout_add_layer_norm_backward(one, 8, 0, one, 8, 0, dh, lddh, 4, 8, one, one, null, 0, 0.1, 1, 2,
                                                       null, dx, dr, null, null, null, 0, null)

    assert addb(dx=null, dr=null) == -1 and addb(lddh=7) == -1 and addb(dh=ctypes.c_void_p(18)) == -1
    assert lib.m3d_layer_norm_workspace_bytes(0, 8, 0) > 0 and lib.m3d_layer_norm_workspace_bytes(100, 64, 1) >= 2 * 64 * 4


def test_modules_without_a_gpu():
    ref = torch.nn.LayerNorm(24)
    torch.nn.init.normal_(ref.weight)
    m = layers.LayerNorm(24)
    m.load_state_dict(ref.state_dict())
    assert torch.equal(m.weight, ref.weight) and layers.LayerNorm(24, affine=False).weight is None
    with pytest.raises(ValueError, match="features"):
        layers.LayerNorm(0)
    x = torch.randn(3, 24)
    assert layers.dropout(x, 0.5, training=False) is x and layers.dropout(x, 0.0) is x
    assert layers.Dropout(0.4).eval()(x) is x
    torch.manual_seed(3)
    a, b = layers.Dropout(0.4), layers.Dropout(0.4)
    assert not torch.equal(a.rng, b.rng) and a.state_dict()["rng"].tolist() == a.rng.tolist()
    assert layers.Dropout(0.4, seed=9).rng.tolist() == [9, 0]


def test_layer_norm_backbone_is_built_and_refused_by_the_engine():
    kw = dict(channels=(32, 64, 64, 32), layers=(1, 1, 1, 1), out_channels=32)
    net = spunet.SpUNet(norm="layer", dropout=0.1, **kw)
    plain = spunet.SpUNet(**kw)
    skip = ("running_mean", "running_var", "num_batches_tracked", "rng")
    names = lambda m: {k for k in m.state_dict() if not k.endswith(skip)}
    assert names(net) == names(plain)
    blocks = [m for m in net.modules() if isinstance(m, spunet.PDLayerNorm)]
    assert blocks and all(m.drop.p == 0.1 for m in blocks)
    with pytest.raises(ValueError, match="unknown norm"):
        spunet.SpUNet(norm="group", **kw)
    with pytest.raises(ValueError, match="needs norm"):
        spunet.SpUNet(dropout=0.1, **kw)
    from segmentation_amd import engine
    sd = {"backbone." + k: v for k, v in net.state_dict().items()}
    with pytest.raises(ValueError, match="batch-norm statistics"):
        engine._fold_norm(sd, "backbone.conv_input.bn", 0, torch.zeros(1, 256))
    one = spunet.SpUNet(norm="layer", norm_decouple=False, norm_adaptive=False, **kw)
    with pytest.raises(ValueError, match="batch-norm statistics"):
        engine._fold_norm(one.state_dict(), "conv_input.bn", 0, None)
