"""Linear layers in 8-bit integers for passes without a gradient (csrc/gemm_i8.hip): an evaluation, or a teacher's forward.

    quantize_rows(x)                                   (int8 [..., K], float32 [...]): one scale per row
    linear_int8(x, weight, weight_scale, bias, relu)   the layer: x is quantised per token, the sums are 32-bit integers
    Int8Linear                                         an nn.Linear's weights held that way, one scale per output channel
    quantize_ffn_(module)                              puts Int8Linear in the place of every FFN's two linears

Rounding is to nearest, ties to even, of the exact quotient 127 x / max|x|; the integer sums are exact, so a result does not
depend on the batch a token comes in."""
from __future__ import annotations

import torch

from . import _native

MAX_K = 131072


def _rows(x: torch.Tensor) -> torch.Tensor:
    x2 = x if x.dim() == 2 else x.reshape(x.numel() // x.shape[-1], x.shape[-1])
    if x2.stride(1) != 1 or (x2.shape[0] > 1 and x2.stride(0) < x2.shape[1]):
        x2 = x2.contiguous()
    return x2


def _check_float(x: torch.Tensor, what: str) -> None:
    if x.dtype not in _native.DTYPE:
        raise TypeError(f"{what}: float32, float16 or bfloat16, got {x.dtype}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{what}: rows of at least one element, got {tuple(x.shape)}")
    if x.shape[-1] > MAX_K:
        raise NotImplementedError(f"{what}: rows of at most {MAX_K} elements, got {x.shape[-1]}")


def _quantize(x2: torch.Tensor):
    """x2 [rows, K] -> (int8 [rows, bytes] with zeros behind column K, float32 [rows])."""
    rows, K = x2.shape
    q = torch.empty(rows, int(_native.lib.datr_quantized_row_bytes(K)), dtype=torch.int8, device=x2.device)
    scale = torch.empty(rows, dtype=torch.float32, device=x2.device)
    with _native.on_device(x2.device):
        rc = _native.lib.datr_quantize_rows_i8(_native.DTYPE[x2.dtype], x2.data_ptr(), rows, K, max(x2.stride(0), K), q.data_ptr(),
                                               q.shape[1], scale.data_ptr(), _native.current_stream_ptr(x2.device))
    _native.check(rc, "quantize_rows_i8")
    return q, scale


def quantize_rows(x: torch.Tensor):
    """x [..., K] -> (q int8 [..., K], scale float32 [...]) with x ~ q * scale[..., None]: scale = max|x| / 127 over the row; x is
    taken as a constant.  A row of zeros has scale 0; a row with an infinity or a NaN has scale NaN (and q 0).  q's rows are held
    at a distance of a multiple of 256 bytes, the layout that `linear_int8` reads without a copy."""
    _check_float(x, "quantize_rows")
    if not x.is_cuda:
        raise RuntimeError("quantize_rows: Not implemented on the CPU")
    K = x.shape[-1]
    q, scale = _quantize(_rows(x.detach()))
    return q[:, :K].view(x.shape), scale.view(x.shape[:-1])


def linear_int8(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, bias: torch.Tensor = None, relu: bool = False,
                out_dtype: torch.dtype = None) -> torch.Tensor:
    """relu?(x W^T + bias) with x [..., K] quantised per token and W = weight * weight_scale[:, None]: weight int8 [N, K],
    weight_scale float32 [N], bias float32 [N] or None -> [..., N] in `out_dtype` (x's by default).

    Weight rows that start at 16-byte borders (`quantize_rows` holds them so) are read as they are; others are copied on every
    call.  A token with an infinity or a NaN gives a row of NaN.  No gradient: x must not require one."""
    _check_float(x, "linear_int8")
    if out_dtype is None:
        out_dtype = x.dtype
    elif out_dtype not in _native.DTYPE:
        raise TypeError(f"linear_int8: the result is float32, float16 or bfloat16, got {out_dtype}")
    if weight.dtype is not torch.int8 or weight_scale.dtype is not torch.float32 or (bias is not None and bias.dtype is not torch.float32):
        raise TypeError("linear_int8: weight is int8, weight_scale and bias are float32")
    lead, K = x.shape[:-1], x.shape[-1]
    if weight.dim() != 2 or weight.shape[1] != K:
        raise ValueError(f"linear_int8: weight {tuple(weight.shape)} does not fit rows of {K}")
    N = weight.shape[0]
    if weight_scale.shape != (N,) or (bias is not None and bias.shape != (N,)):
        raise ValueError(f"linear_int8: weight_scale and bias have {N} entries")
    if torch.is_grad_enabled() and (x.requires_grad or weight_scale.requires_grad or (bias is not None and bias.requires_grad)):
        raise RuntimeError("linear_int8 has no gradient: call it under torch.no_grad(), or detach its inputs")
    if _native.carries_tangent(x) or _native.carries_tangent(weight_scale) or (bias is not None and _native.carries_tangent(bias)):
        raise RuntimeError("linear_int8 has no gradient, in forward mode either")
    if not x.is_cuda:
        raise RuntimeError("linear_int8: Not implemented on the CPU")
    device = x.device
    if weight.device != device or weight_scale.device != device or (bias is not None and bias.device != device):
        raise ValueError("linear_int8: x, weight, weight_scale and bias are on different devices")
    apart, step = weight.stride()
    if step != 1 or apart % 16 or apart < K or weight.data_ptr() % 16:
        held = torch.empty((N, -(-K // 16) * 16), dtype=torch.int8, device=device)[:, :K]
        weight, apart = held.copy_(weight), held.stride(0)
    if not weight_scale.is_contiguous():
        weight_scale = weight_scale.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    x2 = _rows(x)
    M = x2.shape[0]
    y = torch.empty((*lead, N), dtype=out_dtype, device=device)
    need = _native.lib.datr_linear_i8_workspace_bytes(M, K)
    ws = torch.empty(need, dtype=torch.int8, device=device) if need else None
    with _native.on_device(device):
        rc = _native.lib.datr_linear_i8(
            _native.DTYPE[x.dtype], x2.data_ptr(), max(x2.stride(0), K), weight.data_ptr(), apart, weight_scale.data_ptr(),
            0 if bias is None else bias.data_ptr(), M, N, K, 1 if relu else 0, _native.DTYPE[out_dtype], y.data_ptr(), N,
            0 if ws is None else ws.data_ptr(), need, _native.current_stream_ptr(device))
    _native.check(rc, "linear_i8")
    return y


class Int8Linear(torch.nn.Module):
    """An nn.Linear's weights as int8 with one scale per output channel; no parameters, no gradient.  The scales and the bias are
    float32 and stay so when the model is cast; the result has x's type."""

    def __init__(self, linear: torch.nn.Linear):
        super().__init__()
        self.in_features, self.out_features = linear.in_features, linear.out_features
        q, scale = quantize_rows(linear.weight.detach())
        self.register_buffer("weight", q)
        self.register_buffer("weight_scale", scale)
        self.register_buffer("bias", None if linear.bias is None else linear.bias.detach().float().clone())

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs):
        weight, scale = state_dict.get(prefix + "weight"), state_dict.get(prefix + "weight_scale")
        if weight is not None and weight.dtype is not torch.int8:
            # a cast would leave zeros; an error stops the load whatever `strict` says
            error_msgs.append(f"{prefix}weight is int8 with a scale per row, got {weight.dtype}: load a float checkpoint before the layer "
                              "is quantised")
        elif (weight is None) != (scale is None):
            error_msgs.append(f"{prefix}weight and {prefix}weight_scale belong together, got one of them")
        else:
            super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs)
            self._hold_rows()
            self._keep_float32(self.weight_scale, self.bias)              # (assigned from a checkpoint in half precision)

    def _hold_rows(self) -> None:
        """Rows at 16-byte borders: a move to another device and an assigned checkpoint pack them, and linear_int8 would copy them
        on every call.  Not in forward: a buffer bound anew inside a graph's capture, on one of two streams or under inference
        mode is not what the next call may use."""
        if self.weight.stride(0) % 16 or self.weight.stride(1) != 1:
            held = torch.empty((self.out_features, -(-self.in_features // 16) * 16), dtype=torch.int8, device=self.weight.device)
            self.weight = held[:, :self.in_features].copy_(self.weight)

    def _keep_float32(self, scale, bias) -> None:
        # half() and its like cast a model's float buffers; the layer reads these two in 32 bits whatever x is
        for name, before in (("weight_scale", scale), ("bias", bias)):
            now = getattr(self, name)
            if now is not None and now.dtype is not torch.float32:
                setattr(self, name, before.to(now.device, torch.float32))

    def _apply(self, fn, recurse=True):
        scale, bias = self.weight_scale, self.bias
        super()._apply(fn, recurse)
        self._hold_rows()
        self._keep_float32(scale, bias)
        return self

    def forward(self, x: torch.Tensor, relu: bool = False) -> torch.Tensor:
        return linear_int8(x, self.weight, self.weight_scale, self.bias, relu=relu)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"


def quantize_ffn_(module: torch.nn.Module) -> int:
    """Replaces `linear1` and `linear2` of every encoder / decoder layer below `module` (an evaluation model or a frozen
    teacher on its device) by Int8Linear, in place; returns how many layers were changed.  The rest of the model keeps its
    precision: the feed-forward products are over half of a forward pass' matrix work.

    A teacher that takes EMA updates stays in floats: datr_amd.ema refuses 8-bit layers, so quantise a deepcopy of it after
    each update."""
    changed = 0
    for layer in list(module.modules()):
        pair = [getattr(layer, name, None) for name in ("linear1", "linear2")]
        if all(isinstance(p, torch.nn.Linear) for p in pair):
            layer.linear1, layer.linear2 = Int8Linear(pair[0]), Int8Linear(pair[1])
            changed += 1
    return changed
