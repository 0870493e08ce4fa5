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
derivatives of tanh and sigmoid that of a byte.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from muzero_amd import _hip
from muzero_amd._hip import ptr
from muzero_amd._rows import TYPE, check_tensor, on_device, row_stride, rows_of, stream_of, workspace
from muzero_amd.quantized import ACTIVATIONS, QuantizedRows, quantize_rows


def save_activations(x: torch.Tensor) -> QuantizedRows:
    """x [..., K] as an 8-bit checkpoint (scales of three significant bits).  `.dequantize()` reads it back."""
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
    dz = rows_of(dz.detach())
    (R, N), K = dz.shape, saved.columns
    make = torch.empty if R > 0 else torch.zeros
    dw = make((N, K), dtype=dz.dtype, device=dz.device)
    db = make(N, dtype=dz.dtype, device=dz.device) if want_bias else None
    if R > 0:
        lib, kind = _hip.lib(), TYPE[dz.dtype]
        with on_device(dz):
            need = lib.mz_ckpt8_workspace(kind, saved.scale_bits, R, N, K)
            ws = workspace(need, dz)
            _hip.check(lib.mz_ckpt8_weight_grad(ptr(dz), kind, row_stride(dz), R, N, ptr(saved.codes), saved.ld,
                                                ptr(saved.scales), saved.scale_bits, K, ptr(dw), K, ptr(db), ptr(ws), need,
                                                stream_of(dz)), "mz_ckpt8_weight_grad")
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


class _CheckpointedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, activation):
        y = _activate_(F.linear(x, weight, bias), activation)
        codes = scales = act = None
        if y.numel() > 0:
            if ctx.needs_input_grad[1]:
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
    fewer (nothing is kept under torch.no_grad())."""
    check_tensor(x, "x")
    check_tensor(weight, "weight")
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1] or x.shape[-1] < 1:
        raise ValueError(f"x of shape {tuple(x.shape)} does not match a weight of shape {tuple(weight.shape)}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {ACTIVATIONS}, not {activation!r}")
    if not torch.is_grad_enabled():
        return _activate_(F.linear(x, weight, bias), activation)
    return _CheckpointedLinear.apply(x, weight, bias, activation)


class eight_bit_checkpoints:
    """Context manager: inside it the dense layers of the given networks -- every build_mlp sequence and the merge layer
    of a DynamicsNetwork -- keep 8-bit checkpoints on the GPU.  Convolutions and BatchNorm layers are left as they are,
    and so is everything on the CPU.  Parameters, state_dict keys and results of the forward pass do not change."""

    def __init__(self, *modules: torch.nn.Module):
        from muzero_amd.neural_networks.network_builder import is_dense_sequence
        self.sequences = [m for net in modules for m in net.modules() if is_dense_sequence(m)]
        self.merges = [m for net in modules for m in net.modules() if hasattr(m, "fc_merge") and hasattr(m, "merge")]
        self._patched: list[tuple[torch.nn.Module, str]] = []

    @staticmethod
    def _sequence_forward(seq, x):
        from muzero_amd.neural_networks.network_builder import dense_pairs
        if not x.is_cuda:
            return torch.nn.Sequential.forward(seq, x)
        for lin, act in dense_pairs(seq):
            if act == "softmax":
                x = torch.softmax(checkpointed_linear(x, lin.weight, lin.bias), dim=1)
            else:
                x = checkpointed_linear(x, lin.weight, lin.bias, act)
        return x

    @staticmethod
    def _merge(net, merged):
        if not merged.is_cuda:
            return type(net).merge(net, merged)
        return checkpointed_linear(merged, net.fc_merge.weight, net.fc_merge.bias, "relu")

    def __enter__(self):
        for mods, name, fn in ((self.sequences, "forward", self._sequence_forward), (self.merges, "merge", self._merge)):
            for m in mods:
                if name not in m.__dict__:  # an outer context of the same kind has done it already
                    m.__dict__[name] = (lambda x, _m=m, _f=fn: _f(_m, x))
                    self._patched.append((m, name))
        return self

    def __exit__(self, *exc):
        while self._patched:
            m, name = self._patched.pop()
            del m.__dict__[name]
        return False
