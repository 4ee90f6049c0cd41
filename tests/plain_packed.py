"""A plain restatement of the 4-bit cache in float64 on the CPU: where its codes lie, what they stand for, how a value gets its code, and
attention over it.  Written from the layout's description, element by element through index maps."""

from __future__ import annotations

import math

import torch

F64 = torch.float64


def places(hd: int):
    """For keys and for values [16, hd]: a code's byte and shift, and the bytes of its step and offset, in a block of 20 * hd bytes."""
    ng = hd // 32
    p, d = torch.meshgrid(torch.arange(16), torch.arange(hd), indexing="ij")
    j, c = d // 32, d % 32
    key_nibble = p * hd + 8 * ((c // 8) * ng + j) + c % 8
    key_step = 8 * hd + p * 4 * ng + 2 * j
    h, t, u = p // 8, p % 8 // 2, p % 2
    value_nibble = 8 * (((h * 8 + c // 4) * 4 + t) * ng + j) + 4 * u + c % 4
    value_step = 18 * hd + (p // 2) * 8 * ng + 4 * j + 2 * u
    return ((key_nibble // 2, 4 * (key_nibble % 2), key_step, key_step + 2 * ng),
            (10 * hd + value_nibble // 2, 4 * (value_nibble % 2), value_step, value_step + 4 * ng))


def _bf16_at(blocks: torch.Tensor, at: torch.Tensor) -> torch.Tensor:
    bits = (blocks[..., at].int() << 16) | (blocks[..., at + 1].int() << 24)
    return bits.view(torch.float32).to(F64)


def read(blocks: torch.Tensor):
    """Blocks [..., 20 * hd] -> for keys and for values (codes, steps, offsets), each [..., 16, hd]."""
    out = []
    for byte, shift, step, offset in places(blocks.shape[-1] // 20):
        out.append(((blocks[..., byte] >> shift.to(torch.uint8)) & 15, _bf16_at(blocks, step), _bf16_at(blocks, offset)))
    return out


def values(blocks: torch.Tensor):
    """Keys and values [..., 16, hd] in float64."""
    return [offset + step * codes.to(F64) for codes, step, offset in read(blocks)]


def bf16_toward(x: torch.Tensor, up: bool) -> torch.Tensor:
    """float64 values rounded up or down to bfloat16 ones (float64 again)."""
    near = x.to(torch.float32).to(torch.bfloat16)
    wrong = near.to(F64) < x if up else near.to(F64) > x
    return torch.where(wrong, torch.nextafter(near, torch.full_like(near, math.inf if up else -math.inf)), near).to(F64)


def quantise(x: torch.Tensor):
    """(codes, steps, offsets) of x [..., hd], each [..., hd], by the definition."""
    groups = x.to(F64).unflatten(-1, (-1, 32))
    offset = bf16_toward(groups.amin(-1), False).unsqueeze(-1)
    step = bf16_toward((groups.amax(-1, keepdim=True) - offset) / 15, True)
    codes = torch.where(step > 0, torch.round((groups - offset) / step), 0.0).clamp(0, 15)
    return codes.flatten(-2), step.expand_as(codes).flatten(-2), offset.expand_as(codes).flatten(-2)


def pack(k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
    """Keys and values [..., 16, hd] as blocks [..., 20 * hd]."""
    hd = k.shape[-1]
    blocks = torch.zeros((*k.shape[:-2], 20 * hd), dtype=torch.uint8)
    for x, (byte, shift, step_at, offset_at) in zip((k, v), places(hd)):
        codes, step, offset = quantise(x)
        flat = blocks.view(-1, 20 * hd)
        n = flat.shape[0]
        flat.scatter_add_(1, byte.reshape(1, -1).expand(n, -1), (codes.to(torch.uint8) << shift.to(torch.uint8)).reshape(n, -1))
        for at, param in ((step_at, step), (offset_at, offset)):
            bits = param.reshape(n, -1).to(torch.float32).view(torch.int32) >> 16
            flat[:, at.reshape(-1)] = (bits & 255).to(torch.uint8)
            flat[:, at.reshape(-1) + 1] = (bits >> 8 & 255).to(torch.uint8)
    return blocks


def attention(q, keys, vals, pos, scale, window=0, chunk=0, sinks=None, softcap=0.0, rounded=False):
    """One row: q [tokens, nh, hd] at positions ``pos``; keys and values as (codes, steps, offsets), [positions, nkv, hd] each.
    Returns the result [tokens, nh, hd] in float64, and how far a kernel may be from it.

    The bound, with u = 2^-8 the most that a rounding to bfloat16 moves a value: the result is rounded, u |o|.  The single tokens'
    kernel rounds a group's weights step p for codes that count from 8, and weights p for offset + 8 step: u sum p (|code - 8| step +
    |offset + 8 step|).  A prompts' kernel (``rounded``) rounds p and the values: 2 u sum p |v| (or less:
    half precision's u is an eighth).  A score that is off by d moves
    every weight by a factor of at most e^(2 d): 2 d (1 + d) sum p |v| more.  d, in a prompts' kernel: keys are rounded to half precision
    (times 2^-6), u / 8 |k| or 2^-19, and sums are added up in float32 (40 roundings of 2^-23).  Else: a query channel is off by at most
    2^-17 of the head's largest (two parts of 4 bits of a value scaled to 128 .. 256, the second on a grid of 2^-9), which a code multiplies
    by up to 15 steps, and sums of up to 32 terms and of groups are added up in float32, 40 roundings of at most 2^-23 of what is summed,
    codes and offsets apart."""
    group = q.shape[1] // keys[0].shape[1]
    (kc, ks, ko), (vc, vs, vo) = ([x.to(F64).repeat_interleave(group, dim=1) for x in part] for part in (keys, vals))
    k, v = ko + ks * kc, vo + vs * vc
    s = torch.einsum("thd,khd->htk", q, k) * scale
    if rounded:
        d = torch.einsum("thd,khd->htk", q.abs(), k.abs() * (2.0 ** -11 + 40 * 2.0 ** -23) + 2.0 ** -19) * abs(scale)
        weight = 2 * v.abs()
    else:
        d = torch.einsum("thd,khd->htk", q.abs(), ks * kc + ko.abs()) * 40 * 2.0 ** -23
        d = abs(scale) * (d + 15 * 2.0 ** -17 * q.abs().amax(-1).T.unsqueeze(-1) * ks.sum(-1).T.unsqueeze(1))
        weight = (vc - 8).abs() * vs + (vo + 8 * vs).abs()
    d = d + 2.0 ** -20 * (1 + s.abs())
    if softcap:
        s = softcap * torch.tanh(s / softcap)
        d = d + 2.0 ** -20 * softcap
    key = torch.arange(k.shape[0])
    pos = pos.view(1, -1, 1)
    hidden = key > pos
    if window:
        hidden |= key <= pos - window
    if chunk:
        hidden |= key < pos // chunk * chunk
    s = s.masked_fill(hidden, -math.inf)
    d = d.masked_fill(hidden, 0.0).amax(-1, keepdim=True).permute(1, 0, 2)
    if sinks is not None:
        sink = sinks.to(F64).view(-1, 1, 1).expand(-1, s.shape[1], 1)
        p = torch.softmax(torch.cat([s, sink], -1), -1)[..., :-1]
    else:
        p = torch.softmax(s, -1)
    o = torch.einsum("htk,khd->thd", p, v)
    u = 2.0 ** -8
    return o, u * torch.einsum("htk,khd->thd", p, weight) + 2 * d * (1 + d) * torch.einsum("htk,khd->thd", p, v.abs()) + u * o.abs() + 1e-6
