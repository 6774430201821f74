"""Layer norm, dropout and the residual add that joins them, as differentiable functions and modules over the kernels of
ops.layer_norm_fwd, ops.dropout and ops.dropout_add_layer_norm_fwd: what a transformer block on point features is made
of around its matrix products (nn.LayerNorm and nn.Dropout in mosaic3d/src/models/networks/opensegment3d).

Activations [..., c] in float32, bfloat16 or float16, weight and bias in the same type or float32.  First derivatives
in reverse mode only.  Dropout masks are functions of (seed, offset, row, channel) and are recomputed in the backward pass."""
import torch
import torch.nn as nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import ops


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = ops.layer_norm_fwd(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        dx, dweight, dbias = ops.layer_norm_backward(x, dy, mean, rstd, weight, ctx.needs_input_grad[1],
                                                     ctx.needs_input_grad[2])
        return dx, dweight, dbias, None


class _DropoutFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, offset, state):
        ctx.drop = (p, seed, offset)
        ctx.save_for_backward(state)
        return ops.dropout(x, p, seed, offset, state)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return ops.dropout(dy, *ctx.drop, *ctx.saved_tensors), None, None, None, None


class _DropoutAddLayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps, p, seed, offset, state):
        y, h, mean, rstd = ops.dropout_add_layer_norm_fwd(x, residual, weight, bias, eps, p, seed, offset, state)
        ctx.save_for_backward(h, weight, mean, rstd, state)
        ctx.drop = (p, seed, offset)
        ctx.x_dtype = x.dtype
        ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh):
        h, weight, mean, rstd, state = ctx.saved_tensors
        want = ctx.needs_input_grad
        if dy is None:   # only h was used
            if dh is None:
                return (None,) * 9
            dy = torch.zeros(h.shape, dtype=ctx.x_dtype, device=h.device)
        grads = ops.dropout_add_layer_norm_backward(h, dy, dh, mean, rstd, weight, *ctx.drop, state, *want[:4])
        return (*grads, None, None, None, None, None)


def _taped(*ts):
    """Does autograd follow the call?  Dual tensors of forward-mode differentiation go the same way: the Functions have no
    rule for tangents and say so, where the kernels alone would lose them."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts):
        return True
    return forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in ts)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Layer norm over the last axis (ops.layer_norm_fwd), differentiable in x, weight and bias."""
    if not _taped(x, weight, bias):
        return ops.layer_norm_fwd(x, weight, bias, eps)[0]
    return _LayerNormFn.apply(x, weight, bias, eps)


def _mask_of(x, seed, offset, state):
    """(seed, offset, state) of one call's mask: what was given, or a seed of its own from torch's CPU generator (which
    activation checkpointing restores for the forward that it computes again)."""
    if seed is None and offset is None and state is None:
        if x.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("dropout: a captured call needs a generator state (ops.dropout_next); a seed that is drawn "
                               "on the host would be the same on every replay")
        seed = int(torch.randint(0, 2 ** 62, (), device="cpu"))
    return 0 if seed is None else seed, 0 if offset is None else offset, state


def dropout(x, p=0.5, training=True, seed=None, offset=None, state=None):
    """Dropout (ops.dropout), differentiable in x; x itself outside training or with p = 0.  The mask is a function of
    (seed, offset) or of a `state` (ops.dropout_next); a call that is given none of them draws a seed from torch's
    generator."""
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability {p} is not in [0, 1]")
    if not training or p == 0.0:
        return x
    seed, offset, state = _mask_of(x, seed, offset, state)
    if not _taped(x):
        return ops.dropout(x, p, seed, offset, state)
    return _DropoutFn.apply(x, p, seed, offset, state)


def dropout_add_layer_norm(x, residual, weight=None, bias=None, eps=1e-5, p=0.0, training=True, seed=None,
                           offset=None, state=None, need_h=True):
    """(y, h) with h = residual + dropout(x) and y = layer norm of h (ops.dropout_add_layer_norm_fwd), differentiable in
    x, residual, weight and bias through both outputs; no dropout outside training; the mask as in `dropout`.  The
    residual stream is of x's type or float32.  need_h=False: the caller goes on with y alone (post-norm blocks); h is None
    where no gradient needs it."""
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability {p} is not in [0, 1]")
    if not training or p == 0.0:
        p, seed, offset, state = 0.0, 0, 0, None
    else:
        seed, offset, state = _mask_of(x, seed, offset, state)
    if not _taped(x, residual, weight, bias):
        return ops.dropout_add_layer_norm_fwd(x, residual, weight, bias, eps, p, seed, offset, state, need_h)[:2]
    return _DropoutAddLayerNormFn.apply(x, residual, weight, bias, eps, p, seed, offset, state)


class LayerNorm(nn.Module):
    """nn.LayerNorm over the last axis: same parameter names, so its state dict loads unchanged."""

    def __init__(self, num_features, eps=1e-5, affine=True):
        super().__init__()
        if not 1 <= num_features <= ops.LAYER_NORM_MAX_CHANNELS:
            raise ValueError(f"LayerNorm: 1 to {ops.LAYER_NORM_MAX_CHANNELS} features, got {num_features}")
        self.num_features, self.eps, self.affine = int(num_features), float(eps), affine
        self.weight = nn.Parameter(torch.ones(num_features)) if affine else None
        self.bias = nn.Parameter(torch.zeros(num_features)) if affine else None

    def forward(self, x):
        return layer_norm(x, self.weight, self.bias, self.eps)

    def extra_repr(self):
        return f"{self.num_features}, eps={self.eps}, affine={self.affine}"


class Dropout(nn.Module):
    """Dropout whose generator state is a buffer `rng` (seed, offset) on the module's device: it is saved with the
    model, and a captured graph draws a new mask on every replay.  Without a seed one is drawn from torch's generator;
    ranks that shall draw different masks are given different seeds.  Every call in training moves the state on; a
    forward that is computed twice for one backward pass (activation checkpointing) takes a `state` that the caller
    drew once (`draw`), and a draw inside the recomputation is refused: it would be another mask."""

    def __init__(self, p=0.5, seed=None):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"dropout probability {p} is not in [0, 1]")
        self.p = float(p)
        if seed is None:
            seed = int(torch.randint(0, 2 ** 62, (), device="cpu"))
        # where a module's buffers are made; a generator has a value from the start, also in a module without storage
        device = torch.get_default_device()
        self.register_buffer("rng", ops.dropout_state(seed, "cpu" if device.type == "meta" else device))

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs):
        """A state dict without a generator (of nn.Dropout, or of a model that was trained without dropout) leaves the
        module its own."""
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs)
        if prefix + "rng" in missing_keys:
            missing_keys.remove(prefix + "rng")

    def draw(self):
        """The (seed, offset) of one call, or None where nothing is dropped."""
        if not (self.training and self.p > 0.0):
            return None
        if torch._C._current_graph_task_id() != -1:
            raise RuntimeError("dropout: a mask is drawn inside a backward pass, by a forward that is recomputed "
                               "(activation checkpointing); its gradients would belong to another mask than its result.  "
                               "Draw the state in front of the checkpointed call and hand it in (state=, or "
                               "dropout_states= of SpUNet)")
        return ops.dropout_next(self.rng)

    def forward(self, x, state=None):
        return dropout(x, self.p, self.training, state=self.draw() if state is None else state)

    def extra_repr(self):
        return f"p={self.p}"


class DropoutAddLayerNorm(nn.Module):
    """(x, residual) -> (y, h): h = residual + dropout(x), y = layer norm of h.  `state`: as in Dropout.  Whether values
    are dropped goes by the mode of the `drop` module (`train()` and `eval()` set it with the block's own)."""

    def __init__(self, num_features, p=0.0, eps=1e-5, affine=True, seed=None):
        super().__init__()
        self.norm = LayerNorm(num_features, eps, affine)
        self.drop = Dropout(p, seed)

    def forward(self, x, residual, state=None):
        return dropout_add_layer_norm(x, residual, self.norm.weight, self.norm.bias, self.norm.eps, self.drop.p,
                                      self.drop.training, state=self.drop.draw() if state is None else state)
