"""Dense layers in 8-bit integers: rows with a scale each, and products of them.

    weight = quantize_rows(linear.weight)                 # one scale per output channel, once per weight update
    y = int8_linear(x, weight, linear.bias, "relu")       # rows of x are coded in the call, one scale per row
    heads = Int8MLP(pred_net.policy_mlp)                  # a whole build_mlp sequence

The int8 form of nn.Linear + activation (`build_mlp`, src/neural_networks/network_builder.py:183-205) for networks that
answer with trained weights: a quarter of the weight bytes of float32, the matrix cores' int8 rate.  Values are off by
the two roundings to 127 steps of the largest value of a row, which is NOT the float32 accuracy of the search's own
networks (muzero_amd.engine): choose it where that is enough.
"""
from __future__ import annotations

from typing import Optional

import torch

from muzero_amd import _hip
from muzero_amd._hip import ptr
from muzero_amd._rows import TYPE, check_on_gpu, check_tensor, in_memory, on_device, refuse_tangent, row_stride, rows_of, stream_of, workspace

MAX_K = 131072  # sums of K products of codes stay exact in 32 bits
ACTIVATIONS = ("none", "linear", "relu", "tanh", "sigmoid")


class QuantizedRows:
    """Rows in 8 bits: x[r, k] is about scales[r] * codes[r, k].

    codes       i8[rows, ldc] in -127..127, ldc a multiple of 128, rows on 16-byte addresses; zero behind the last column
    scales      f32[rows]
    shape       of the tensor that was coded
    dtype       of the tensor that was coded, float32, bfloat16 or float16
    scale_bits  significant bits of the scales: 24, or 3 if every one is 1, 1.25, 1.5 or 1.75 times a power of two"""

    __slots__ = ("codes", "scales", "shape", "dtype", "scale_bits")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape, dtype: torch.dtype, scale_bits: int):
        shape = torch.Size(shape)
        if codes.dtype != torch.int8 or codes.dim() != 2 or scales.dtype != torch.float32 or scales.dim() != 1:
            raise TypeError("codes must be an int8 matrix and scales a float32 vector")
        if codes.device != scales.device:
            raise ValueError(f"codes are on {codes.device}, scales on {scales.device}")
        if dtype not in TYPE:
            raise TypeError(f"rows are of float32, bfloat16 or float16, not {dtype}")
        if scale_bits not in (24, 3):
            raise ValueError(f"scale_bits must be 24 or 3, not {scale_bits}")
        rows, ldc = codes.shape
        if len(shape) < 1 or not 1 <= shape[-1] <= ldc or rows != shape[:-1].numel() or scales.shape[0] != rows:
            raise ValueError(f"codes of shape {tuple(codes.shape)} and {scales.shape[0]} scales do not hold a tensor of shape {tuple(shape)}")
        if ldc % 128 or codes.data_ptr() % 16 or not scales.is_contiguous() or codes.stride(1) != 1 or (
                rows > 1 and (codes.stride(0) % 128 or codes.stride(0) < ldc)):
            raise ValueError("codes need rows of a multiple of 128 adjacent bytes on 16-byte addresses, scales adjacent values")
        self.codes, self.scales, self.shape, self.dtype, self.scale_bits = codes, scales, shape, dtype, scale_bits

    @classmethod
    def _of(cls, codes, scales, shape, dtype, scale_bits) -> "QuantizedRows":
        """Without the checks, for codes this package has laid out itself."""
        q = object.__new__(cls)
        q.codes, q.scales, q.shape, q.dtype, q.scale_bits = codes, scales, shape, dtype, scale_bits
        return q

    @property
    def rows(self) -> int:
        return self.codes.shape[0]

    @property
    def columns(self) -> int:
        return self.shape[-1]

    @property
    def ld(self) -> int:
        """Bytes from one row of codes to the next."""
        return self.codes.stride(0) if self.codes.shape[0] > 1 else self.codes.shape[1]

    def dequantize(self, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """scales * codes in the shape and (by default) the type of the tensor that was coded."""
        dtype = self.dtype if dtype is None else dtype
        if dtype not in TYPE:
            raise TypeError(f"rows can be read back as float32, bfloat16 or float16, not {dtype}")
        check_on_gpu(self.codes, "codes")
        out = torch.empty(self.shape, dtype=dtype, device=self.codes.device)
        if self.rows > 0:
            with on_device(out):
                _hip.check(_hip.lib().mz_dequant8_rows(ptr(self.codes), self.ld, ptr(self.scales), self.rows, self.columns, ptr(out),
                                                       TYPE[dtype], self.columns, stream_of(out)), "mz_dequant8_rows")
        return out


def quantize_rows(x: torch.Tensor, scale_bits: int = 24) -> QuantizedRows:
    """Codes of x [..., K], one scale per row.  scale_bits=3 rounds the scale up to 1, 1.25, 1.5 or 1.75 times a power of
    two (what muzero_amd.checkpoints keeps).  Codes are whole numbers and carry no gradient; an x with a forward-mode tangent
    is refused."""
    check_tensor(x, "x")
    if scale_bits not in (24, 3):
        raise ValueError(f"scale_bits must be 24 or 3, not {scale_bits}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x needs at least one value in a row, not shape {tuple(x.shape)}")
    rows = rows_of(x.detach() if x.requires_grad else x)
    (R, K), dev = rows.shape, rows.device
    ldc = (K + 127) // 128 * 128
    codes = torch.empty((R, ldc), dtype=torch.int8, device=dev)
    scales = torch.empty(R, dtype=torch.float32, device=dev)
    if R > 0:
        with on_device(rows):
            rc = _hip.lib().mz_quant8_rows(rows.data_ptr(), TYPE[rows.dtype], row_stride(rows), R, K, scale_bits, codes.data_ptr(),
                                           ldc, scales.data_ptr(), stream_of(rows))
            if rc:
                _hip.check(rc, "mz_quant8_rows")
    return QuantizedRows._of(codes, scales, x.shape, x.dtype, scale_bits)


def _check_weight(weight: QuantizedRows, K: int) -> int:
    if not isinstance(weight, QuantizedRows):
        raise TypeError("weight must be the QuantizedRows of a [N, K] matrix (quantize_rows)")
    if len(weight.shape) != 2:
        raise ValueError(f"weight must be a matrix, not of shape {tuple(weight.shape)}")
    if weight.columns != K:
        raise ValueError(f"rows of {K} values do not match a weight of {weight.columns} input features")
    if K > MAX_K:
        raise ValueError(f"{K} input features are more than the {MAX_K} whose sums stay exact in 32 bits")
    return weight.rows


def int8_linear(x, weight: QuantizedRows, bias: Optional[torch.Tensor] = None, activation: str = "none",
                out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """act(x W^T + bias) for x [..., K] (a tensor, or QuantizedRows when several layers read the same rows).  The result
    has x's type unless `out_dtype` says otherwise.  There is no gradient, reverse or
    forward mode: training goes through float weights (muzero_amd.checkpoints keeps their inputs in 8 bits)."""
    coded = isinstance(x, QuantizedRows)
    if not coded:
        check_tensor(x, "x")
        if x.dim() < 1:
            raise ValueError("x needs at least one dimension")
        if torch.is_grad_enabled() and x.requires_grad:
            raise RuntimeError("int8_linear has no gradient; call it under torch.no_grad() or on a detached tensor")
    N = _check_weight(weight, x.shape[-1])
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {ACTIVATIONS}, not {activation!r}")
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if out_dtype not in TYPE:
        raise TypeError(f"out_dtype must be float32, bfloat16 or float16, not {out_dtype}")
    dev = weight.codes.device
    if (x.codes if coded else x).device != dev:
        raise ValueError("x and weight are on different devices")
    if bias is not None:
        if bias.shape != (N,) or bias.device != dev:
            raise ValueError(f"bias must be {N} values on {dev}")
        refuse_tangent(bias, "bias")
        if bias.dtype is not torch.float32 or not bias.is_contiguous() or bias.is_neg():
            bias = in_memory(bias.detach().to(torch.float32))
    check_on_gpu(weight.codes, "weight")
    K = weight.columns
    y = torch.empty(x.shape[:-1] + (N,), dtype=out_dtype, device=dev)
    if y.numel() == 0:
        return y
    lib, act = _hip.lib(), _hip.ACT[activation]
    with on_device(y):
        if coded:
            need = lib.mz_int8_codes_workspace(x.rows, K, N)
            ws = workspace(need, y)
            _hip.check(lib.mz_int8_forward_codes(ptr(x.codes), x.ld, ptr(x.scales), x.rows, K, ptr(weight.codes),
                                                 weight.ld, ptr(weight.scales), N, ptr(bias), act, ptr(y), TYPE[out_dtype],
                                                 N, ptr(ws), need, stream_of(y)), "mz_int8_forward_codes")
        else:
            rows = rows_of(x)
            R = rows.shape[0]
            need = lib.mz_int8_workspace(R, K, N)
            ws = workspace(need, y)
            rc = lib.mz_int8_forward(rows.data_ptr(), TYPE[rows.dtype], row_stride(rows), R, K, weight.codes.data_ptr(), weight.ld,
                                     weight.scales.data_ptr(), N, ptr(bias), act, y.data_ptr(), TYPE[out_dtype], N, ptr(ws), need,
                                     stream_of(y))
            if rc:
                _hip.check(rc, "mz_int8_forward")
    return y


def _renew(old, new):
    """`new` in the memory of `old`, where that fits."""
    if old is None or new is None or old.shape != new.shape:
        return new
    if isinstance(new, QuantizedRows):
        old.codes.copy_(new.codes), old.scales.copy_(new.scales)
    else:
        old.copy_(new)
    return old


class Int8MLP:
    """A build_mlp sequence (Linear + activation pairs) with its weights in 8 bits.  Call `refresh()` after the weights
    change: it writes the new codes where the old ones are, so recorded graphs go on with them.  `logits(x)` stops in
    front of a final softmax."""

    def __init__(self, seq: torch.nn.Sequential, device="cuda"):
        self.seq, self.device = seq, torch.device(device)
        self.layers, self.softmax = [], False
        self.refresh()

    def refresh(self) -> None:
        from muzero_amd.neural_networks.network_builder import dense_pairs
        pairs = dense_pairs(self.seq)
        if any(act == "softmax" for _, act in pairs[:-1]):
            raise ValueError("softmax is supported as the last activation only")
        self.softmax = pairs[-1][1] == "softmax"
        old = self.layers if len(self.layers) == len(pairs) else [(None, None, None)] * len(pairs)
        self.layers = [(_renew(w, quantize_rows(lin.weight.detach().to(self.device))),
                        None if lin.bias is None else _renew(b, lin.bias.detach().to(self.device, torch.float32, copy=True)),
                        "none" if act == "softmax" else act) for (w, b, _), (lin, act) in zip(old, pairs)]

    def logits(self, x) -> torch.Tensor:
        for w, b, act in self.layers:
            x = int8_linear(x, w, b, act)
        return x

    def __call__(self, x) -> torch.Tensor:
        y = self.logits(x)
        return self.seq[-1](y) if self.softmax else y


class Int8Networks:
    """Device evaluator of a (g, f) pair without residual blocks whose dense layers are in 8-bit integers: what
    `muzero_amd.engine.make_networks(g, f, int8=True)` returns, for `BatchedMCTS` in lock step (the single-launch search is
    written for the float32-accurate networks).  Meant for wide layers, where a search is bound by the weights it reads.

    g merges per latent, not per child: fc_merge of [latent ; embedding] is its latent half in 8 bits, once for the A
    children of a node, plus the float32 row of the action (mz_action_table; src/neural_networks/neural_network.py:168-172).
    Call `refresh()` after the weights change."""

    fusable = False
    strided_outputs = True    # results may go to strided columns; the A children of a node share one row index

    def __init__(self, dynamics: torch.nn.Module, prediction: torch.nn.Module, device="cuda"):
        if len(dynamics.res_blocks) or len(prediction.res_blocks) or not isinstance(dynamics.res_final, torch.nn.Identity) \
                or not isinstance(prediction.res_final, torch.nn.Identity):
            raise NotImplementedError("8-bit networks cover res_net: [] configurations")
        self.device = torch.device(device)
        self.dynamics_net, self.prediction_net = dynamics, prediction
        c, h, w = dynamics.latent_shape
        self.D, self.A = c * h * w, dynamics.num_actions
        self.heads = [Int8MLP(m, device) for m in (dynamics.reward_mlp, prediction.value_mlp, prediction.policy_mlp)]
        self.merge = None
        self.table = torch.empty((self.A, self.D), dtype=torch.float32, device=self.device)
        self._merge()

    def refresh(self) -> None:
        for head in self.heads:
            head.refresh()
        self._merge()

    def _merge(self) -> None:
        from muzero_amd.neural_networks.network_builder import is_plain
        g, D, A = self.dynamics_net, self.D, self.A
        if not is_plain(g.fc_merge, torch.nn.Linear):
            raise ValueError("fc_merge must be a Linear layer without hooks or a forward of its own")
        emb, w, b = (t.detach().to(self.device, torch.float32).contiguous()
                     for t in (g.action_embedding.weight, g.fc_merge.weight, g.fc_merge.bias))
        self.merge = _renew(self.merge, quantize_rows(w[:, :D]))
        with on_device(self.table):
            _hip.check(_hip.lib().mz_action_table(ptr(emb), ptr(w), ptr(b), D, A, ptr(self.table), stream_of(self.table)),
                       "mz_action_table")

    def _rows(self, latent: torch.Tensor, B: int, rows: Optional[torch.Tensor]) -> torch.Tensor:
        """Latent rows [B, D]; a negative index names a row of zeros."""
        flat = latent.reshape(-1, self.D)
        if rows is None:
            return flat[:B]
        picked = flat[rows.clamp(min=0).long()]
        return torch.where((rows >= 0)[:, None], picked, torch.zeros((), device=picked.device))

    @torch.no_grad()
    def dynamics(self, latent, B, *, ld=None, rows=None, action=None, next_latent=None, ld_next=None, next_rows=None, reward=None) -> None:
        A = self.A
        U = B if action is not None else B // A
        base = int8_linear(self._rows(latent, U, rows), self.merge)
        if action is not None:
            nxt = (base + self.table[action.long()]).relu_()
        else:
            nxt = (base[:, None, :] + self.table).relu_().reshape(B, self.D)
        if reward is not None:
            (reward.view(B) if reward.is_contiguous() else reward).copy_(self.heads[0](nxt)[:, 0])
        if next_latent is not None:
            out = next_latent.view(-1, self.D)
            if next_rows is None:
                out[:B] = nxt
            else:  # rows below 0 are skipped
                if next_rows.dtype == torch.int64:  # what 32 bits do not hold names no row
                    next_rows = next_rows.clamp(-1, (1 << 31) - 1)
                next_rows = next_rows.reshape(-1).to(torch.int32).contiguous()
                if next_rows.numel() != B or next_rows.device != nxt.device:
                    raise ValueError(f"next_rows must be {B} rows on {nxt.device}")
                if out.dtype != torch.float32 or out.device != nxt.device or (self.D > 1 and out.stride(1) != 1):
                    raise ValueError(f"next_latent must be float32 with adjacent values in a row, on {nxt.device}")
                with on_device(nxt):
                    _hip.check(_hip.lib().mz_scatter_rows(ptr(nxt), self.D, ptr(next_rows), B, self.D, ptr(out), row_stride(out),
                                                          out.shape[0], stream_of(nxt)), "mz_scatter_rows")

    @torch.no_grad()
    def prediction(self, latent, B, *, ld=None, rows=None, softmax_times=0, policy=None, value=None, argmax=None) -> None:
        x = quantize_rows(self._rows(latent, B, rows))     # both heads read the same rows
        if value is not None:
            value.copy_(self.heads[1](x)[:, 0])
        if policy is None and argmax is None:
            return
        probs = self.heads[2].logits(x)
        lib, A = _hip.lib(), self.A
        with on_device(probs):
            st = stream_of(probs)
            _hip.check(lib.mz_policy_post(ptr(probs), B, A, 1, ptr(probs), None, st), "mz_policy_post")
            out = probs if softmax_times == 0 else torch.empty_like(probs)
            _hip.check(lib.mz_policy_post(ptr(probs), B, A, softmax_times, ptr(out), ptr(argmax), st), "mz_policy_post")
        if policy is not None:
            policy.copy_(out)
