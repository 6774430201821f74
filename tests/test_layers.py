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


# ---------------------------------------------------------------- modules over stand-ins of the kernels' definitions
@pytest.fixture
def definitions(monkeypatch):
    """ops.* of this family on the CPU, from the float64 formulas and the generator's definition; `calls` of the dropout
    functions: (p, seed, offset, state)."""
    calls = []

    def keep(x, p, seed, offset, state):
        calls.append((p, seed, offset, None if state is None else state.tolist()))
        if state is not None:
            seed, offset = int(state[0]), offset + int(state[1])
        n, c = x.numel() // x.shape[-1], x.shape[-1]
        return O.dropout(torch.ones(n, c, dtype=torch.float64), p, seed, offset).reshape(x.shape)

    def next_state(state, step=1):
        used = state.clone()
        state[1] += step
        return used

    def drop(x, p, seed=0, offset=0, state=None):
        return (x.double() * keep(x, p, seed, offset, state)).to(x.dtype)

    def norm(x, weight=None, bias=None, eps=1e-5):
        y, mean, rstd = O.layer_norm(x.double(), weight, bias, eps)
        return y.to(x.dtype).detach(), mean.detach(), rstd.detach()

    def norm_back(x, dy, mean, rstd, weight=None, want_dweight=True, want_dbias=True):
        dx, dw, db = O.layer_norm_backward(x.double(), dy.double(), mean, rstd, weight)
        return dx.to(x.dtype), dw.to(x.dtype) if want_dweight else None, db.to(x.dtype) if want_dbias else None

    def add(x, residual, weight=None, bias=None, eps=1e-5, p=0.0, seed=0, offset=0, state=None, want_h=True):
        h = (residual.double() + x.double() * keep(x, p, seed, offset, state)).to(residual.dtype)
        y, mean, rstd = norm(h, weight, bias, eps)
        return y.to(x.dtype), h.detach() if want_h else None, mean, rstd

    def add_back(h, dy, dh, mean, rstd, weight=None, p=0.0, seed=0, offset=0, state=None, want_dx=True,
                 want_dresidual=True, want_dweight=True, want_dbias=True):
        t, dw, db = norm_back(h, dy, mean, rstd, weight, want_dweight, want_dbias)
        t = t if dh is None else t + dh
        dx = (t.double() * keep(t, p, seed, offset, state)).to(dy.dtype)
        return dx if want_dx else None, t if want_dresidual else None, dw, db

    for name, fn in (("dropout", drop), ("dropout_next", next_state), ("layer_norm_fwd", norm),
                     ("layer_norm_backward", norm_back), ("dropout_add_layer_norm_fwd", add),
                     ("dropout_add_layer_norm_backward", add_back)):
        monkeypatch.setattr(ops, name, fn)
    return calls


@pytest.mark.parametrize("reentrant", [False, True])
def test_a_recomputed_forward_does_not_draw(definitions, reentrant):
    """Under activation checkpointing a module that draws for itself is refused; a state that was drawn in front of the
    call gives the gradients of the plain call, and the generator moves on once."""
    from torch.utils.checkpoint import checkpoint
    torch.manual_seed(1)
    x, r = torch.randn(20, 16, requires_grad=True), torch.randn(20, 16, requires_grad=True)
    gy = torch.randn(20, 16)
    norm = spunet.PDLayerNorm(16, 4, dropout=0.5)
    block, drop = layers.DropoutAddLayerNorm(16, 0.5, seed=3), layers.Dropout(0.5, seed=4)
    forms = [(norm.drop, lambda a, b, st: norm(a, "ScanNet", residual=b, relu=True, state=st)),
             (block.drop, lambda a, b, st: block(a, b, st)[0]),
             (drop, lambda a, b, st: drop(a, st) + b)]
    for module, form in forms:
        y = checkpoint(lambda a, b: form(a, b, None), x, r, use_reentrant=reentrant)
        with pytest.raises(RuntimeError, match="inside a backward pass"):
            (y * gy).sum().backward()
        before = module.rng.clone()
        st = module.draw()
        want = torch.autograd.grad((form(x, r, st) * gy).sum(), (x, r))
        x.grad = r.grad = None
        (checkpoint(lambda a, b: form(a, b, st), x, r, use_reentrant=reentrant) * gy).sum().backward()
        assert torch.equal(x.grad, want[0]) and torch.equal(r.grad, want[1]) and want[0].abs().sum() > 0
        assert module.rng.tolist() == [before[0].item(), before[1].item() + 1]
        x.grad = r.grad = None
        (form(x, r, None) * gy).sum().backward()   # a plain call draws its own, in front of its backward pass
    norm.eval()
    assert torch.equal(norm(x, "ScanNet", residual=r, state=st), norm(x, "ScanNet", residual=r))
    assert "_state" not in norm.__dict__


def test_network_states_are_drawn_and_counted():
    kw = dict(channels=(32, 64, 64, 32), layers=(1, 1, 1, 1), out_channels=32)
    net = spunet.SpUNet(norm="layer", dropout=0.1, **kw)
    blocks = [m for m in net.modules() if isinstance(m, spunet.BasicBlock)]
    assert net._dropping_norms() == [b.bn2 for b in blocks] and len(blocks) == 4
    assert net.eval().draw_dropout() == [None] * 4
    assert spunet.SpUNet(norm="layer", **kw).draw_dropout() == [] and spunet.SpUNet(**kw).draw_dropout() == []
    with pytest.raises(ValueError, match="drops in 4 blocks"):
        net(dict(dropout_states=[None] * 3))
    with pytest.raises(ValueError, match="drops in 0 blocks"):
        spunet.SpUNet(**kw)(dict(dropout_states=[None]))


@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(definitions, monkeypatch, grad):
    """Forward-mode differentiation has no rule here; the call says so, whichever argument carries the tangent, and a call
    without tangents inside the same level runs."""
    import torch.autograd.forward_ad as fw
    for name in ("layer_norm_fwd", "dropout", "dropout_add_layer_norm_fwd"):   # raw addresses carry no tangent
        fn = getattr(ops, name)
        monkeypatch.setattr(ops, name, lambda *a, fn=fn: fn(*(t.detach() if isinstance(t, torch.Tensor) else t for t in a)))
    x, w = torch.randn(4, 8), torch.ones(8)
    with torch.set_grad_enabled(grad), fw.dual_level():
        d, dw = fw.make_dual(x, torch.ones_like(x)), fw.make_dual(w, torch.ones_like(w))
        for call in (lambda: layers.layer_norm(d), lambda: layers.layer_norm(x, dw, w), lambda: layers.dropout(d, 0.5, seed=1),
                     lambda: layers.dropout_add_layer_norm(d, x), lambda: layers.dropout_add_layer_norm(x, d, w, w),
                     lambda: layers.dropout_add_layer_norm(x, x, w, dw)):
            with pytest.raises(NotImplementedError, match="jvp"):
                call()
        layers.layer_norm(x, w, w), layers.dropout_add_layer_norm(x, x, w, w, p=0.5, seed=1), layers.dropout(x, 0.5, seed=1)
    assert torch.equal(layers.layer_norm(x, w, w), O.layer_norm(x.double(), w, w)[0].float())
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.jvp(layers.layer_norm, (x,), (x,))


def test_the_dropout_of_a_block_goes_by_its_own_mode(definitions):
    """A block whose dropout alone was switched off drops nothing; one whose dropout alone is on draws a mask a call."""
    calls = definitions
    x = torch.randn(6, 8)
    block = layers.DropoutAddLayerNorm(8, 0.5, seed=7)
    block.drop.eval()
    assert torch.equal(block(x, x)[1], 2 * x) and calls[-1] == (0.0, 0, 0, None)
    assert torch.equal(block(x, x, ops.dropout_state(1, "cpu"))[1], 2 * x) and block.drop.rng.tolist() == [7, 0]
    block.eval()
    block.drop.train()
    h0, h1 = block(x, x)[1], block(x, x)[1]
    assert calls[-2:] == [(0.5, 0, 0, [7, 0]), (0.5, 0, 0, [7, 1])] and not torch.equal(h0, h1)
    block.train()
    block(x, x)
    assert calls[-1] == (0.5, 0, 0, [7, 2])
    block.eval()
    assert torch.equal(block(x, x)[1], 2 * x) and block.drop.rng.tolist() == [7, 3]


def test_dropout_seed_of_the_network():
    """Networks of one dropout_seed drop alike, those of another differ in every block; blocks differ among themselves;
    the seed leaves torch's generator and the parameters as they are."""
    kw = dict(channels=(32, 64, 64, 32), layers=(1, 1, 1, 1), out_channels=32, norm="layer", dropout=0.1)
    nets = []
    for seed in (0, 0, 1, None):
        torch.manual_seed(2)
        nets.append(spunet.SpUNet(dropout_seed=seed, **kw))
    seeds = [[m.rng[0].item() for m in net.modules() if isinstance(m, layers.Dropout)] for net in nets]
    assert seeds[0] == seeds[1] and not set(seeds[0]) & set(seeds[2]) and not set(seeds[0]) & set(seeds[3])
    assert all(len(set(s)) == len(s) for s in seeds)
    assert all(m.rng[1] == 0 for m in nets[0].modules() if isinstance(m, layers.Dropout))
    assert all(torch.equal(p, q) for p, q in zip(nets[0].parameters(), nets[2].parameters()))


def test_functions_without_a_seed_draw_one(definitions):
    """As torch's own dropout: two calls drop different values, torch's generator repeats them, and a recomputed forward
    gets its first mask again.  What names a seed, an offset or a state has that mask."""
    from torch.utils.checkpoint import checkpoint
    calls = definitions
    x = torch.randn(12, 16, requires_grad=True)
    both = lambda t, **kw: (layers.dropout(t, 0.5, **kw), layers.dropout_add_layer_norm(t, t, p=0.5, **kw)[1])
    torch.manual_seed(4)
    a, b = both(x), both(x)
    torch.manual_seed(4)
    again = both(x)
    for u, v, w in zip(a, b, again):
        assert not torch.equal(u, v) and torch.equal(u, w)
    for kw, seen in ((dict(seed=0), (0, 0, None)), (dict(offset=3), (0, 3, None)), (dict(offset=0), (0, 0, None)),
                     (dict(seed=5, offset=6), (5, 6, None)), (dict(state=torch.tensor([8, 9])), (0, 0, [8, 9]))):
        before = torch.get_rng_state()
        both(x, **kw)
        assert calls[-1] == calls[-2] == (0.5, *seen) and torch.equal(before, torch.get_rng_state())
    before = torch.get_rng_state()
    assert layers.dropout(x, 0.0) is x and layers.dropout(x, 0.5, False) is x
    layers.dropout_add_layer_norm(x, x), layers.dropout_add_layer_norm(x, x, p=0.5, training=False)
    assert torch.equal(before, torch.get_rng_state())
    for reentrant in (False, True):
        torch.manual_seed(5)
        want = torch.autograd.grad(both(x)[0].square().sum(), x)[0]
        torch.manual_seed(5)
        x.grad = None
        checkpoint(lambda t: both(t)[0], x, use_reentrant=reentrant).square().sum().backward()
        assert torch.equal(x.grad, want) and want.abs().sum() > 0


def test_state_dicts_with_and_without_generators():
    """Strict loads both ways between a network with dropout and one without, a resumed generator, and a state dict of
    nn.Dropout; other keys are as strict as before."""
    kw = dict(channels=(32, 64, 64, 32), layers=(1, 1, 1, 1), out_channels=32, norm="layer")
    with_drop, bare = spunet.SpUNet(dropout=0.1, dropout_seed=1, **kw), spunet.SpUNet(**kw)
    twin = spunet.SpUNet(dropout=0.3, dropout_seed=2, **kw)
    sd = with_drop.state_dict()
    sd["enc.0.block0.bn2.drop.rng"][1] = 40
    bare.load_state_dict(sd)
    assert all(torch.equal(p, q) for p, q in zip(bare.parameters(), with_drop.parameters()))
    seed = twin.enc[0].block0.bn2.drop.rng.clone()
    twin.load_state_dict(bare.state_dict())
    assert torch.equal(twin.enc[0].block0.bn2.drop.rng, seed)
    twin.load_state_dict(sd)
    assert twin.enc[0].block0.bn2.drop.rng.tolist() == sd["enc.0.block0.bn2.drop.rng"].tolist()
    drop = layers.Dropout(0.2, seed=6)
    drop.load_state_dict(torch.nn.Dropout(0.2).state_dict())
    assert drop.rng.tolist() == [6, 0]
    for bad in (dict(sd, extra=seed), {k: v for k, v in sd.items() if k != "enc.0.block0.bn2.bns.0.weight"},
                {**sd, "enc.0.block0.bn2.drop.other": seed}):
        for net in (twin, bare):
            with pytest.raises(RuntimeError, match="key"):
                net.load_state_dict(bad)


def test_modules_under_a_default_device():
    """Constructed without storage (to be filled by load_state_dict(assign=True)), a module still has a generator."""
    with torch.device("meta"):
        block = layers.DropoutAddLayerNorm(8, 0.5)
        seeded = layers.Dropout(0.5, seed=12)
    assert block.norm.weight.is_meta and block.drop.rng.device.type == "cpu" and seeded.rng.tolist() == [12, 0]
    source = layers.DropoutAddLayerNorm(8, 0.5, seed=3)
    block.load_state_dict(source.state_dict(), assign=True)
    assert not block.norm.weight.is_meta and block.drop.rng.tolist() == [3, 0]
    kw = dict(channels=(32, 64, 64, 32), layers=(1, 1, 1, 1), out_channels=32, norm="layer", dropout=0.1, dropout_seed=3)
    here = spunet.SpUNet(**kw)
    with torch.device("meta"):
        there = spunet.SpUNet(**kw)
    assert torch.equal(there.enc[0].block0.bn2.drop.rng, here.enc[0].block0.bn2.drop.rng)
