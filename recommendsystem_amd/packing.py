"""8-bit activation checkpoints (rs_pack8 / rs_unpack8): what a layer keeps of an activation for its
backward pass, in a quarter (fp32) or half (bf16, fp16) of the memory.

    pack8(x)                       [..., D] -> codes int8 [..., D], scales fp32 [..., ceil(D / 128)]
    unpack8(codes, scales, dtype)  the values they stand for

Each block of 128 columns of a row has one scale, max|x| / 127, and every code is x / scale to the
nearest whole number: a value is kept to within max|x| / 254 of its block.  Blocks with max|x| <
2^-100 come back as zeros; an infinity or NaN comes back as NaN in all of its block.

`layers.Dense(save_8bit=True)` and `sequence.layer_norm(save_8bit=True)` keep their inputs so.
"""
from __future__ import annotations

import torch

from ._lib import call, device_index, empty, empty_as, run_on

BLOCK = 128
ELEMENT_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def element_code(t: torch.Tensor, what: str) -> int:
    code = ELEMENT_TYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{what} must be float32, bfloat16 or float16, got {t.dtype}")
    return code


def rows_of(t: torch.Tensor) -> torch.Tensor:
    """t [..., D] as a 2-D view with unit column stride, in place where its strides allow it."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _width(x: torch.Tensor, what: str) -> int:
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{what} needs a last dimension of at least 1, got shape {tuple(x.shape)}")
    if x.shape[-1] > 2 ** 30:
        raise ValueError(f"{what}: a last dimension of {x.shape[-1]} is not supported")
    return x.shape[-1]


def scale_shape(shape) -> tuple:
    return (*shape[:-1], -(-shape[-1] // BLOCK))


def pack8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of x [..., D] float32 / bfloat16 / float16 (any strides).  Not a
    differentiable operation: the codes are kept, not computed with."""
    D = _width(x, "pack8")
    code = element_code(x, "pack8's input")
    return run_on(device_index(x), _pack, x.detach(), D, code)


def _pack(x, D, code, stream):
    x2 = rows_of(x)
    codes, scales = empty_as(x, torch.int8), empty(scale_shape(x.shape))
    call("rs_pack8", stream, code, x2.data_ptr(), x2.stride(0), x2.shape[0], D, codes.data_ptr(),
         scales.data_ptr())
    return codes, scales


def unpack8(codes: torch.Tensor, scales: torch.Tensor, dtype=torch.float32) -> torch.Tensor:
    """The values of pack8's pair, as a contiguous tensor of codes' shape."""
    D = _width(codes, "unpack8")
    if codes.dtype != torch.int8 or scales.dtype != torch.float32:
        raise TypeError(f"unpack8 takes int8 codes and float32 scales, got {codes.dtype} and {scales.dtype}")
    if tuple(scales.shape) != scale_shape(codes.shape):
        raise ValueError(f"unpack8: scales {tuple(scales.shape)} do not fit codes {tuple(codes.shape)} "
                         f"(expected {scale_shape(codes.shape)})")
    if dtype not in ELEMENT_TYPES:
        raise TypeError(f"unpack8: dtype must be float32, bfloat16 or float16, got {dtype}")
    return run_on(device_index(codes, scales), _unpack, codes, scales, D, dtype)


def _unpack(codes, scales, D, dtype, stream):
    codes, scales = codes.contiguous(), scales.contiguous()
    y = empty_as(codes, dtype)
    call("rs_unpack8", stream, ELEMENT_TYPES[dtype], codes.data_ptr(), scales.data_ptr(),
         codes.numel() // D, D, y.data_ptr(), D)
    return y
