"""8-bit activation checkpoints: what a dense layer keeps for its backward pass, in a quarter of the bytes.

`nn.Linear` keeps its input for the weight gradient and its activation's output for the derivative, in full.  Here the
input is kept as row codes (one byte per value, a scale per row) and the activation as one bit (relu) or one byte
(tanh, sigmoid) per value; the weight gradient is formed from the codes without writing the input out again:

    y = checkpointed_linear(x, layer.weight, layer.bias, "relu")   # one layer
    with eight_bit_checkpoints(dyn_net, pred_net):                 # the dense layers of whole networks
        policy, value = pred_net(latent)
    learner = DataParallelLearner(..., checkpoints8=True)          # the unroll of src/training.py:244-305

Results of the forward pass are unchanged.  The gradient that goes on to the input is exact for relu and linear layers;
weight gradients carry the codes' rounding (half a step of at most 1.25 / 127 of a row's largest value), and the
derivatives of tanh and sigmoid that of a byte: tanh is kept to half a step of 1 / 127, so the derivative is off by up to
0.008, and a unit beyond +-126.5 / 127 (a sigmoid below 0.002 or above 0.998) has no gradient at all.
"""
from __future__ import annotations

import threading
import types
from typing import Optional

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from muzero_amd import _hip
from muzero_amd._hip import ptr
from muzero_amd._rows import TYPE, check_tensor, on_device, refuse_tangent, row_stride, rows_of, stream_of, workspace
from muzero_amd.quantized import ACTIVATIONS, QuantizedRows, quantize_rows


MAX_CHECKPOINT_ROWS = 1 << 20  # that one weight gradient takes


def save_activations(x: torch.Tensor) -> QuantizedRows:
    """x [..., K] as an 8-bit checkpoint (scales of three significant bits).  `.dequantize()` reads it back.

    The short scale makes the products of a 16-bit gradient exact in fewer planes.  For a float32 gradient it saves nothing:
    weight_grad takes `quantize_rows(x)`, whose steps are up to a fifth smaller, in the same time."""
    return quantize_rows(x, scale_bits=3)


def weight_grad(dz: torch.Tensor, saved: QuantizedRows, want_bias: bool = True):
    """(dW [N, K], db [N] or None) of a layer z = x W^T + b from dz [..., N] and the checkpoint of x [..., K], in dz's
    type: dW = dz^T x, db = the column sums of dz."""
    check_tensor(dz, "dz")
    if not isinstance(saved, QuantizedRows):
        raise TypeError("saved must be what save_activations returned")
    if dz.dim() < 1 or dz.shape[-1] < 1 or dz.shape[:-1] != saved.shape[:-1]:
        raise ValueError(f"dz of shape {tuple(dz.shape)} does not match a checkpoint of shape {tuple(saved.shape)}")
    if dz.device != saved.codes.device:
        raise ValueError(f"dz is on {dz.device}, the checkpoint on {saved.codes.device}")
    dz = rows_of(dz.detach() if dz.requires_grad else dz)
    (R, N), K = dz.shape, saved.columns
    make = torch.empty if R > 0 else torch.zeros
    dw = make((N, K), dtype=dz.dtype, device=dz.device)
    db = make(N, dtype=dz.dtype, device=dz.device) if want_bias else None
    if R > 0:
        lib, kind = _hip.lib(), TYPE[dz.dtype]
        with on_device(dz):
            need = lib.mz_ckpt8_workspace(kind, saved.scale_bits, R, N, K)
            ws = workspace(need, dz) if need else None
            rc = lib.mz_ckpt8_weight_grad(dz.data_ptr(), kind, row_stride(dz), R, N, saved.codes.data_ptr(), saved.ld,
                                          saved.scales.data_ptr(), saved.scale_bits, K, dw.data_ptr(), K, ptr(db), ptr(ws), need,
                                          stream_of(dz))
            if rc:
                _hip.check(rc, "mz_ckpt8_weight_grad")
    return dw, db


def _act_save(y: torch.Tensor, activation: str) -> torch.Tensor:
    rows = rows_of(y)
    R, N = rows.shape
    act, lib = _hip.ACT[activation], _hip.lib()
    saved = torch.empty((R, lib.mz_ckpt8_act_bytes(N, act)), dtype=torch.uint8, device=y.device)
    with on_device(y):
        _hip.check(lib.mz_ckpt8_act_save(ptr(rows), TYPE[rows.dtype], row_stride(rows), R, N, act, ptr(saved), stream_of(y)),
                   "mz_ckpt8_act_save")
    return saved


def _act_grad(dy: torch.Tensor, saved: torch.Tensor, activation: str) -> torch.Tensor:
    rows = rows_of(dy)
    R, N = rows.shape
    dz = torch.empty((R, N), dtype=dy.dtype, device=dy.device)
    with on_device(dy):
        _hip.check(_hip.lib().mz_ckpt8_act_grad(ptr(rows), TYPE[rows.dtype], row_stride(rows), ptr(saved), R, N,
                                                _hip.ACT[activation], ptr(dz), N, stream_of(dy)), "mz_ckpt8_act_grad")
    return dz


def _activate_(y: torch.Tensor, activation: str) -> torch.Tensor:
    if activation == "relu":
        return y.relu_()
    if activation == "tanh":
        return y.tanh_()
    if activation == "sigmoid":
        return y.sigmoid_()
    return y


def _linear(x, weight, bias):
    """F.linear inside an autograd function.  There autograd is off, and autocast would keep the 16-bit copies it makes of x
    and the parameters for later layers, which would then have no gradient: its cache stays out of this call."""
    if not torch.is_autocast_enabled(x.device.type):
        return F.linear(x, weight, bias)
    cached = torch.is_autocast_cache_enabled()
    torch.set_autocast_cache_enabled(False)
    try:
        return F.linear(x, weight, bias)
    finally:
        torch.set_autocast_cache_enabled(cached)


class _CheckpointedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, activation):
        y = _activate_(_linear(x, weight, bias), activation)
        codes = scales = act = None
        if y.numel() > 0:
            if ctx.needs_input_grad[1]:
                if x.shape[:-1].numel() > MAX_CHECKPOINT_ROWS:
                    raise ValueError(f"{x.shape[:-1].numel()} rows are more than the {MAX_CHECKPOINT_ROWS} of one weight gradient")
                saved = save_activations(x)
                codes, scales = saved.codes, saved.scales
            if activation not in ("none", "linear"):
                act = _act_save(y, activation)
        ctx.save_for_backward(weight if ctx.needs_input_grad[0] else None, codes, scales, act)
        ctx.x_shape, ctx.x_dtype, ctx.w_dtype, ctx.activation = x.shape, x.dtype, weight.dtype, activation
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        refuse_tangent(dy, "the gradient")
        weight, codes, scales, act = ctx.saved_tensors
        K, N = ctx.x_shape[-1], dy.shape[-1]
        want_x, want_w, want_b, _ = ctx.needs_input_grad
        dx = dw = db = None
        dz = rows_of(dy) if act is None else _act_grad(dy, act, ctx.activation)
        if want_x:
            dx = (dz @ weight.to(dz.dtype)).reshape(ctx.x_shape).to(ctx.x_dtype)
        if codes is not None:
            saved = QuantizedRows._of(codes, scales, torch.Size((codes.shape[0], K)), ctx.x_dtype, 3)
            dw, db = weight_grad(dz, saved, want_bias=want_b)
            dw, db = dw.to(ctx.w_dtype), None if db is None else db.to(ctx.w_dtype)
        else:
            if want_w:
                dw = torch.zeros((N, K), dtype=ctx.w_dtype, device=dy.device)
            if want_b:
                db = dz.sum(0, dtype=torch.float32).to(ctx.w_dtype)
        return dx, dw, db, None


def checkpointed_linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                        activation: str = "none") -> torch.Tensor:
    """act(x W^T + bias) for x [..., K], with everything the backward pass needs of x and of the result kept in 8 bits or
    fewer (nothing is kept under torch.no_grad()).  At most 2^20 rows where the weight wants a gradient."""
    check_tensor(x, "x", forward_mode=True)  # torch's own operators serve one under no_grad, the autograd function refuses it
    check_tensor(weight, "weight", forward_mode=True)
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1] or x.shape[-1] < 1:
        raise ValueError(f"x of shape {tuple(x.shape)} does not match a weight of shape {tuple(weight.shape)}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {ACTIVATIONS}, not {activation!r}")
    if not torch.is_grad_enabled():
        return _activate_(F.linear(x, weight, bias), activation)
    return _CheckpointedLinear.apply(x, weight, bias, activation)


def _bound(fn, module):
    return types.MethodType(fn, module)


class _Taken:
    """Stands in for a module's method (`forward`, `merge`) while contexts are open.  Copies and pickles of the module get
    the method itself: they belong to no context."""

    stands_in = True

    def __init__(self, module: torch.nn.Module, name: str, fn):
        self.module, self.name, self.fn, self.depth, self.before = module, name, fn, 0, module.__dict__.get(name)

    def __call__(self, *args, **kwargs):
        return self.fn(self.module, *args, **kwargs)

    def __reduce__(self):
        return _bound, (getattr(type(self.module), self.name), self.module)


def _keeps_8_bits(x: torch.Tensor) -> bool:
    """Whether a layer inside a context keeps x in 8 bits; else it runs as it is.  Hooks that torch calls for every module
    see a layer only if it runs as it is."""
    return x.is_cuda and x.dtype in TYPE and x.shape[:-1].numel() <= MAX_CHECKPOINT_ROWS and not torch.nn.modules.module._has_any_global_hook()


_LOCK = threading.Lock()  # of every module's open contexts


class eight_bit_checkpoints:
    """Context manager: inside it the dense layers of the given networks -- every build_mlp sequence and the merge layer
    of a DynamicsNetwork -- keep 8-bit checkpoints on the GPU.  Convolutions and BatchNorm layers are left as they are, and
    so are layers with hooks or a forward of their own, calls with more than 2^20 rows, everything on the CPU or in float64,
    and the part of a sequence that somebody else runs (PredictionNetwork.policy_logits).  Parameters, state_dict keys and
    results of the forward pass do not change.  Contexts may be nested and overlap: a layer is as it was when the last one
    that names it has ended, except for a forward that somebody has given it meanwhile, which stays."""

    def __init__(self, *modules: torch.nn.Module):
        from muzero_amd.neural_networks.network_builder import is_dense_sequence, is_plain
        from muzero_amd.neural_networks.neural_network import DynamicsNetwork
        self.sequences = [m for net in modules for m in net.modules() if is_dense_sequence(m)]
        self.merges = [m for net in modules for m in net.modules() if isinstance(m, DynamicsNetwork) and
                       type(m).merge is DynamicsNetwork.merge and is_plain(m.fc_merge, torch.nn.Linear)]
        self._open: list[list[_Taken]] = []

    @staticmethod
    def _sequence_forward(seq, input):  # by the name it has in torch
        from muzero_amd.neural_networks.network_builder import dense_pairs
        pairs = dense_pairs(seq, strict=False) if _keeps_8_bits(input) else None
        if pairs is None:  # a hook may have come since the context was opened
            return type(seq).forward(seq, input)
        x = input
        for i, (lin, act) in enumerate(pairs):
            if act == "softmax":
                x = seq[2 * i + 1](checkpointed_linear(x, lin.weight, lin.bias))
            else:
                x = checkpointed_linear(x, lin.weight, lin.bias, act)
        return x

    @staticmethod
    def _merge(net, merged):
        from muzero_amd.neural_networks.network_builder import is_plain
        if not _keeps_8_bits(merged) or not is_plain(net.fc_merge, torch.nn.Linear):
            return type(net).merge(net, merged)
        return checkpointed_linear(merged, net.fc_merge.weight, net.fc_merge.bias, "relu")

    def __enter__(self):
        taken = []
        with _LOCK:
            kinds = ((self.sequences, "forward", self._sequence_forward), (self.merges, "merge", self._merge))
            for m, name, fn in ((m, name, fn) for mods, name, fn in kinds for m in mods):
                own = m.__dict__.get(name)
                if isinstance(own, types.MethodType) and own.__func__ is getattr(type(m), name):
                    own = None
                if own is None:
                    m.__dict__[name] = own = _Taken(m, name, fn)
                if isinstance(own, _Taken):  # anything else is somebody's own method: left alone
                    own.depth += 1
                    taken.append(own)
            self._open.append(taken)
        return self

    def __exit__(self, *exc):
        with _LOCK:
            for t in self._open.pop():
                t.depth -= 1
                if t.depth > 0 or t.module.__dict__.get(t.name) is not t:  # still in use, or no longer in the method's place
                    continue
                if t.before is None:
                    del t.module.__dict__[t.name]
                else:
                    t.module.__dict__[t.name] = t.before
        return False
