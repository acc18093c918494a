"""Linears with 4-bit weights and group scales (C ABI wrapper).

``Int4Linear`` holds codes 0 .. 15, an fp16 scale per row and group of 32, 64 or
128 columns and, if wanted, a zero point per group (8 otherwise): a weight is
scale * (code - zero).  It stands beside the Block-RVQ linears where a plain
format is wanted, first of all as the vocabulary projection of a stack
(``LlamaStack.quantize_head``), and as the linears of a whole stack
(``llama.int4_llama``).  It is made for decoding: a call reads the weight once for
every 32 tokens, so from about 32 tokens on a dense linear is faster (2048 tokens of a
prompt through 128256 x 4096: 13.8 ms, dense bf16 1.4).  No counterpart in the reference.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch import Tensor, nn

from . import _abi
from .kv8 import _call

GROUP_SIZES = (32, 64, 128)
_BUFFERS = {"packed": torch.uint8, "scales": torch.float16, "zeros": torch.uint8, "bias": torch.bfloat16}


def quantize_int4(weight: Tensor, group_size: int = 128, *, zero_points: bool = False) -> tuple[Tensor, Tensor, Optional[Tensor]]:
    """Codes uint8 [N, K], scales fp16 [N, K / group_size] and zero points (uint8, or None) of a weight [N, K].

    Without zero points a group's scale is its largest magnitude over 7.5 rounded
    to fp16; with them it spans the group's range, zero included.  Codes are the nearest
    ones for the rounded scale.
    """
    N, K = weight.shape
    if group_size not in GROUP_SIZES or K % group_size:
        raise ValueError(f"group_size must be one of {GROUP_SIZES} and divide in_features ({K}), got {group_size}")
    w = weight.float().reshape(N, K // group_size, group_size)
    if not bool(torch.isfinite(w).all()):
        raise ValueError("weight is not finite")
    if zero_points:
        lo, hi = w.amin(-1).clamp(max=0.0), w.amax(-1).clamp(min=0.0)
        scale = (hi - lo) / 15.0
    else:
        scale = w.abs().amax(-1) / 7.5
    scale = scale.clamp(max=65504.0).to(torch.float16)
    step = torch.where(scale > 0, scale.float(), 1.0)
    zero = (-lo / step).round().clamp(0, 15) if zero_points else torch.full_like(step, 8.0)
    codes = (w / step[..., None] + zero[..., None]).round_().clamp_(0, 15).to(torch.uint8).reshape(N, K)
    return codes, scale, zero.to(torch.uint8) if zero_points else None


class Int4Linear(nn.Module):
    """y = x W^T (+ bias), W = scales * (codes - zeros) in groups of columns.

    codes: uint8 [N, K], 0 .. 15; scales: fp16 [N, K / group_size]; zeros: uint8
    like scales, 0 .. 15, or None (8); all on one CUDA device, where they are
    packed once.  bias is kept in bf16; casts of the module change none of this.
    """

    def __init__(self, codes: Tensor, scales: Tensor, zeros: Optional[Tensor] = None, bias: Optional[Tensor] = None):
        super().__init__()
        if codes.dtype != torch.uint8 or codes.dim() != 2:
            raise ValueError("codes must be uint8 [out_features, in_features]")
        N, K = (int(v) for v in codes.shape)
        if scales.dtype != torch.float16 or scales.dim() != 2 or scales.shape[0] != N or scales.shape[1] < 1 or K % scales.shape[1]:
            raise ValueError("scales must be fp16 [out_features, in_features / group_size]")
        self.group_size = K // int(scales.shape[1])
        if self.group_size not in GROUP_SIZES:
            raise ValueError(f"group_size must be one of {GROUP_SIZES}, got {self.group_size}")
        if zeros is not None and (zeros.dtype != torch.uint8 or zeros.shape != scales.shape):
            raise ValueError("zeros must be uint8 like scales")
        if bias is not None and tuple(bias.shape) != (N,):
            raise ValueError("bias must be [out_features]")
        if not codes.is_cuda or any(t is not None and t.device != codes.device for t in (scales, zeros, bias)):
            raise ValueError("Int4Linear packs its weights on the GPU: codes, scales, zeros and bias must be on one CUDA device")
        self.out_features, self.in_features = N, K
        lib = _abi.load()
        nbytes, entries = ctypes.c_size_t(0), ctypes.c_size_t(0)
        _abi.check(lib.wal_int4_packed_size(N, K, self.group_size, ctypes.byref(nbytes), ctypes.byref(entries)),
                   "wal_int4_packed_size")
        dev = codes.device
        self.register_buffer("packed", torch.empty(nbytes.value, dtype=torch.uint8, device=dev))
        self.register_buffer("scales", torch.empty(entries.value, dtype=torch.float16, device=dev))
        self.register_buffer("zeros", None if zeros is None else torch.empty(entries.value, dtype=torch.uint8, device=dev))
        self.register_buffer("bias", None if bias is None else bias.to(torch.bfloat16).contiguous())
        self._layer_cache = None
        codes, scales = codes.contiguous(), scales.contiguous()
        zeros = None if zeros is None else zeros.contiguous()
        with torch.cuda.device(dev):
            st = lib.wal_int4_pack(ctypes.byref(self.layer_struct()), codes.data_ptr(), scales.data_ptr(), _abi.ptr(zeros),
                                   _abi.stream_handle(dev))
        _abi.check(st, "wal_int4_pack")

    @classmethod
    def from_dense(cls, weight: Tensor, group_size: int = 128, *, zero_points: bool = False,
                   bias: Optional[Tensor] = None) -> "Int4Linear":
        """Nearest codes of a dense weight (``quantize_int4``, some rows at a time)."""
        step = max(1, (1 << 27) // max(1, int(weight.shape[1])))
        parts = [quantize_int4(weight[i:i + step], group_size, zero_points=zero_points) for i in range(0, weight.shape[0], step)]
        if not parts:
            raise ValueError("weight has no rows")
        codes, scales = (torch.cat([p[i] for p in parts]) for i in range(2))
        return cls(codes, scales, torch.cat([p[2] for p in parts]) if zero_points else None, bias)

    def layer_struct(self) -> _abi.Int4Layer:
        key = (self.packed.data_ptr(), self.scales.data_ptr(), _abi.ptr(self.zeros), _abi.ptr(self.bias))
        if self._layer_cache is None or self._layer_cache[0] != key:
            self._check_types()
            layer = _abi.Int4Layer(self.out_features, self.in_features, self.group_size, *key)
            self._layer_cache = (key, layer)
        return self._layer_cache[1]

    def __getstate__(self) -> dict:
        return self.__dict__ | {"_layer_cache": None}  # addresses are not copied

    def _check_types(self) -> None:
        for name, dtype in _BUFFERS.items():
            t = getattr(self, name)
            if t is not None and t.dtype != dtype:
                raise ValueError(f"Int4Linear keeps {name} as {dtype}, got {t.dtype}")

    def _apply(self, fn, recurse: bool = True):
        """Moves of the module; casts (``to(dtype)``, ``half``, ..) leave the weight as it is, for the kernels read these types only."""
        def move(t: Tensor) -> Tensor:
            moved = fn(t)
            return moved if moved.dtype == t.dtype else t.to(moved.device)

        return super()._apply(move, recurse)

    def gemv_into(self, x2: Tensor, y: Tensor) -> None:
        """y[M, N] <- x2[M, K] @ W^T (+ bias) on the current stream; x2 bf16 or fp16, y bf16, fp16 or fp32."""
        index, shape, s, o = x2.get_device(), x2.shape, x2.stride(), y.stride()
        M = shape[0] if len(shape) == 2 else 0
        if (index < 0 or shape != (M, self.in_features) or y.shape != (M, self.out_features) or s[1] != 1
                or (o[1] != 1 and self.out_features > 1) or y.get_device() != index or self.packed.get_device() != index):
            raise ValueError(f"x2 [M, {self.in_features}] and y [M, {self.out_features}] must have contiguous rows on the "
                             f"layer's CUDA device ({self.packed.device})")
        if x2.dtype not in (torch.bfloat16, torch.float16) or y.dtype not in _abi.DTYPE_CODE:
            raise ValueError(f"Int4Linear supports bfloat16 and float16 activations (outputs in float32 too), got {x2.dtype}, {y.dtype}")
        if M == 0:
            return
        # the stride of a single row says nothing
        _call(index, "wal_int4_gemv", ctypes.byref(self.layer_struct()), x2.data_ptr(), _abi.DTYPE_CODE[x2.dtype], M,
              s[0] if M > 1 else -(-self.in_features // 8) * 8, y.data_ptr(), o[0] if M > 1 else self.out_features,
              _abi.DTYPE_CODE[y.dtype])

    def forward(self, x: Tensor) -> Tensor:
        if not x.is_cuda:
            raise ValueError("Int4Linear runs on CUDA only (no CPU path); move the input to a CUDA device")
        if x.shape[-1] != self.in_features:
            raise ValueError(f"Feature mismatch: {x.shape[-1]} != {self.in_features}")
        x2 = x.reshape(-1, self.in_features)
        if x2.stride(-1) != 1 or x2.stride(0) % 8 != 0 or x2.stride(0) < self.in_features or x2.data_ptr() % 16 != 0:
            x2 = x2.clone(memory_format=torch.contiguous_format)
        y = torch.empty((x2.shape[0], self.out_features), device=x.device, dtype=x.dtype)
        self.gemv_into(x2, y)
        return y.reshape(*x.shape[:-1], self.out_features)

    def reconstruct_weight(self, out_dtype: torch.dtype = torch.bfloat16) -> Tensor:
        """The dense weight [N, K], scale * (code - zero) rounded once to bf16, fp16 or fp32."""
        if out_dtype not in _abi.DTYPE_CODE:
            raise ValueError(f"reconstruct_weight supports bfloat16, float16 and float32, got {out_dtype}")
        dev = self.packed.device
        if dev.type != "cuda":
            raise ValueError("reconstruct_weight runs on CUDA only; move the module to a CUDA device")
        w = torch.empty((self.out_features, self.in_features), device=dev, dtype=out_dtype)
        with torch.cuda.device(dev):
            st = _abi.load().wal_int4_dequant(ctypes.byref(self.layer_struct()), w.data_ptr(), w.stride(0),
                                              _abi.DTYPE_CODE[out_dtype], _abi.stream_handle(dev))
        _abi.check(st, "wal_int4_dequant")
        return w

    def compressed_bytes(self) -> int:
        """Bytes a call must read for the weight: codes, scales, zero points (+ bias)."""
        groups = self.out_features * (self.in_features // self.group_size)
        total = self.out_features * self.in_features // 2 + groups * (2 if self.zeros is None else 3)
        return total + (0 if self.bias is None else 2 * self.out_features)

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, group_size={self.group_size}, "
                f"zero_points={self.zeros is not None}")
