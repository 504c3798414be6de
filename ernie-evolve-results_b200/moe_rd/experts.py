"""Products of few rows with 4-bit expert weights: the expert layer of a decode step, between ``route_dispatch`` (or
``sort_tokens``) and ``combine`` (or ``unsort_tokens``)."""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _cabi
from ._cabi import ROW_DTYPE
from .sorting import call, check_offsets, check_out, dense, device_index, refuse_tangents, wants_grad, written


class W4Weights(NamedTuple):
    """4-bit weights in the layout of the kernel (see ``moe_rd_expert_matvec_w4`` in include/moe_rd.h)."""
    packed: torch.Tensor           # [E, ceil(N/32), ceil(K/128), 2048] uint8
    scales: torch.Tensor           # [E, ceil(N/32), K/group, 8, 4] bf16 or fp16
    zeros: Optional[torch.Tensor]  # [E, ceil(N/32), K/group, 8, 2] uint8, two zero points a byte; None: all are 8
    N: int
    K: int
    group: int


def _blocked(t: torch.Tensor) -> torch.Tensor:
    """[E, N, G] per-group values as [E, ceil(N/32), G, 8, 4], zero-padded; outputs r, r + 8, r + 16, r + 24 of a block side
    by side."""
    E, N, G = t.shape
    full = t.new_zeros((E, -(-N // 32) * 32, G))
    full[:, :N] = t
    return full.reshape(E, -1, 4, 8, G).permute(0, 1, 4, 3, 2).contiguous()


def pack_w4(q: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None) -> W4Weights:
    """Lay 4-bit weights out for ``expert_matvec_w4``; done once, when a program loads them (on the CPU or a GPU).

    q: [E, N, K/2] uint8 (or [N, K/2] for one matrix), byte b holding input 2b in its low and 2b+1 in its high four bits;
    scales: [E, N, K/group] bf16 or fp16, the type of the rows that will be multiplied; zeros: uint8 of the same shape,
    0..15, or None for 8.  The weight is (q - zero) * scale.  K must be a multiple of group, group of 32.
    """
    if q.dim() == 2:
        q, scales, zeros = q[None], scales[None], None if zeros is None else zeros[None]
    if q.dtype != torch.uint8 or q.dim() != 3:
        raise TypeError("pack_w4: q must be a uint8 tensor [E, N, K/2]")
    if scales.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError("pack_w4: scales must be bfloat16 or float16")
    E, N, half = q.shape
    K = 2 * half
    if scales.dim() != 3 or scales.shape[:2] != q.shape[:2] or scales.shape[2] < 1 or N < 1 or E < 1 or K < 32:
        raise ValueError("pack_w4: scales must be [E, N, K/group]")
    G = scales.shape[2]
    group = K // G
    if K % G or group % 32:
        raise ValueError(f"pack_w4: {G} scales for {K} inputs: groups must be equal and multiples of 32")
    if zeros is not None:
        if zeros.dtype != torch.uint8 or zeros.shape != scales.shape:
            raise ValueError("pack_w4: zeros must be a uint8 tensor like scales")
        if zeros.numel() and int(zeros.max()) > 15:
            raise ValueError("pack_w4: zero points must be 0..15")
    for t in (scales, zeros):
        if t is not None and t.device != q.device:
            raise ValueError("pack_w4: all tensors must be on one device")
    blocks, chunks = -(-N // 32), -(-K // 128)
    packed = torch.empty((E, blocks, chunks, 2048), dtype=torch.uint8, device=q.device)
    if q.is_cuda:
        q, q_at = dense(q)
        call(q.get_device(), _cabi.lib().moe_rd_pack_w4, E, N, K, q_at, packed.data_ptr())
    else:
        full = q.new_zeros((E, blocks * 32, chunks * 64))
        full[:, :N, :half] = q
        # [E, block, part, output, chunk, word, lane j, byte] -> [E, block, chunk, part, output, j, word, byte]
        r = full.reshape(E, blocks, 4, 8, chunks, 4, 4, 4).permute(0, 1, 4, 2, 3, 6, 5, 7)
        o = packed.view(r.shape)
        o[..., 0] = (r[..., 0] & 15) | ((r[..., 1] & 15) << 4)
        o[..., 1] = (r[..., 2] & 15) | ((r[..., 3] & 15) << 4)
        o[..., 2] = (r[..., 0] >> 4) | (r[..., 1] & 0xF0)
        o[..., 3] = (r[..., 2] >> 4) | (r[..., 3] & 0xF0)
    if zeros is not None:
        z = _blocked(zeros)
        zeros = z[..., 0::2] | (z[..., 1::2] << 4)
    return W4Weights(packed, _blocked(scales), zeros, N, K, group)


def expert_matvec_w4(x: torch.Tensor, weights: W4Weights, offsets: Optional[torch.Tensor] = None, *,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out[r] = W_e x[r] for the rows r of every expert e, with 4-bit weights; [R, N] of the type of x.

    x: [R, K] bf16 or fp16 rows in expert order (``permuted`` / ``rows``), of the type of the scales; offsets: [E+1] int32
    device tensor as ``route_dispatch`` and ``sort_tokens`` return it, or None for one matrix that every row goes
    through.  Rows that no expert has become zero.  Products are added in fp32 and rounded once.

    Meant for few rows per expert (the weights of an expert are read once per eight of its rows, or sixteen where
    there are more than eight per expert on average); right for any number.  For
    inference: a row that requires a gradient is refused.
    """
    if not isinstance(weights, W4Weights):
        raise TypeError("expert_matvec_w4: weights must come from pack_w4")
    done = _cabi.fast.expert_matvec_w4(x, weights, offsets, out)
    if done is not False:
        return out if done is True else done
    packed, scales, zeros, N, K, group = weights
    dtype = x.dtype
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise TypeError("expert_matvec_w4: rows must be bfloat16 or float16")
    if scales.dtype is not dtype:
        raise TypeError("expert_matvec_w4: rows and scales must have one type")
    E, blocks = packed.shape[0], -(-N // 32)
    G = K // group
    if x.dim() != 2 or x.shape[1] != K:
        raise ValueError(f"expert_matvec_w4: rows must be [R, {K}]")
    if (packed.shape != (E, blocks, -(-K // 128), 2048) or packed.dtype is not torch.uint8 or not packed.is_contiguous()
            or scales.shape != (E, blocks, G, 8, 4) or not scales.is_contiguous()
            or (zeros is not None and (zeros.shape != (E, blocks, G, 8, 2) or zeros.dtype is not torch.uint8 or not zeros.is_contiguous()))):
        raise ValueError("expert_matvec_w4: weights are not as pack_w4 returns them")
    if offsets is None:
        if E != 1:
            raise ValueError("expert_matvec_w4: offsets are needed where there is more than one expert")
    else:
        check_offsets("expert_matvec_w4", offsets)
        if offsets.numel() != E + 1:
            raise ValueError(f"expert_matvec_w4: offsets must have {E + 1} elements")
    if wants_grad(x, scales):
        raise RuntimeError("expert_matvec_w4 is for inference and has no gradient: pass detached rows")
    refuse_tangents("expert_matvec_w4", x, scales)
    index = device_index("expert_matvec_w4", x, packed, scales, zeros, offsets)
    x, x_at = dense(x)
    R = x.shape[0]
    weights_at, scales_at = packed.data_ptr(), scales.data_ptr()
    zeros_at = None if zeros is None else zeros.data_ptr()
    offsets_at = None if offsets is None else offsets.data_ptr()
    if out is None:
        result = torch.empty((R, N), dtype=dtype, device=x.device)
        at = result.data_ptr()
    else:
        result = out
        given = [(x_at, x.nbytes), (weights_at, packed.nbytes), (scales_at, scales.nbytes)]
        if zeros is not None:
            given.append((zeros_at, zeros.nbytes))
        if offsets is not None:
            given.append((offsets_at, 4 * E + 4))
        at = check_out("expert_matvec_w4", out, (R, N), dtype, index, given)
    call(index, _cabi.lib().moe_rd_expert_matvec_w4, R, N, K, E, group, ROW_DTYPE[dtype], x_at, weights_at, scales_at, zeros_at, offsets_at, at)
    if out is not None:
        written(out)
    return result
