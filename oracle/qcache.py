"""Decoding over a quantised block cache, in float64 and from the definitions:
codes and scales by search among all of them, attention request by request and
head by head, norms and rotations pair by pair.

Pinned by the codes' own tables (OCP e4m3 without infinities, e2m1), by
``torch.softmax`` and by rotations as complex numbers; no counterpart in the
reference, whose caches are 16-bit.
"""
from __future__ import annotations

import math

import torch

F64 = torch.float64
RUN, LEAST = 32, 16


def code_values(bits):
    """The value of every code (4 bits: 16, 8 bits: 256; NaN where e4m3 has one)."""
    if bits == 4:
        e, m, bias, width = 2, 1, 1, 8
    else:
        e, m, bias, width = 4, 3, 7, 128
    out = []
    for c in range(2 * width):
        mag, sign = c % width, -1.0 if c >= width else 1.0
        ex, frac = mag >> m, mag % (1 << m)
        if bits == 8 and mag == 127:
            out.append(math.nan)
        elif ex == 0:
            out.append(sign * frac / (1 << m) * 2.0 ** (1 - bias))
        else:
            out.append(sign * (1 + frac / (1 << m)) * 2.0 ** (ex - bias))
    assert e + m + 1 == bits
    return torch.tensor(out, dtype=F64)


def quantise(x, bits):
    """x [..., D] -> (values that the codes stand for [..., D], scale bytes [..., D / 32])."""
    runs = x.to(F64).unflatten(-1, (-1, RUN))
    table = code_values(bits)
    table = table[: len(table) // 2]
    table = table[~table.isnan()]                     # magnitudes, ascending with the code
    top = runs.abs().amax(-1)
    limits = table[-1] * 2.0 ** (torch.arange(LEAST, 255, dtype=F64) - 127)
    good = runs.isfinite().all(-1)
    s = LEAST + torch.searchsorted(limits, torch.where(good, top, 0.0))
    y = torch.where(good[..., None], runs, 0.0) * (2.0 ** (127 - s.to(F64)))[..., None]
    a = y.abs()
    hi = torch.searchsorted(table, a).clamp_max(len(table) - 1)
    lo = (hi - 1).clamp_min(0)
    up, down = table[hi] - a, a - table[lo]
    code = torch.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi)
    val = torch.copysign(table[code], y) * (2.0 ** (s.to(F64) - 127))[..., None]
    val = torch.where(good[..., None], val, math.nan)
    return val.flatten(-2), torch.where(good, s, 255).to(torch.uint8)


def cache_values(data, scales):
    """A cache [blocks, G, block, ...] and its scales (None: 16 bits) -> float64 [blocks, G, block, D]."""
    if scales is None:
        return data.to(F64)
    if data.dtype == torch.uint8:
        codes = torch.stack((data % 16, data // 16), -1).flatten(-2).long()
        y = code_values(4)[codes]
    else:
        y = code_values(8)[data.view(torch.uint8).long()]
    s = scales.transpose(2, 3).to(F64)
    mul = torch.where(s == 255, math.nan, 2.0 ** (s - 127))
    return y * mul.repeat_interleave(RUN, -1)


def attention(q, keys, values, tables, lengths, *, starts=None, window=None, softcap=None, slopes=None, gate=None,
              scale=None):
    """keys / values as float64 [blocks, G, block, D] -> (out [R, H, D], sum of weight times |value| (and gate))."""
    r, h, d = q.shape
    blocks, g, block, _ = keys.shape
    columns = tables.shape[1]
    scale = d ** -0.5 if scale is None else scale
    out, size = torch.zeros(r, h, d, dtype=F64), torch.zeros(r, h, d, dtype=F64)
    for i, length in enumerate(lengths):
        lo = max(0, length - columns * block, length - window if window else 0, starts[i] if starts is not None else 0)
        at = [p for p in range(lo, length) if 0 <= int(tables[i, p // block % columns]) < blocks]
        if not at:
            continue
        ids = [int(tables[i, p // block % columns]) for p in at]
        rows = [p % block for p in at]
        back = length - 1 - torch.tensor(at, dtype=F64)
        for head in range(h):
            ks, vs = keys[ids, head // (h // g), rows], values[ids, head // (h // g), rows]
            x = ks @ q[i, head].to(F64) * scale
            if softcap is not None:
                x = softcap * torch.tanh(x / softcap)
            if slopes is not None:
                x = x - slopes[head].to(F64) * back
            w = torch.softmax(x, 0)
            out[i, head], size[i, head] = w @ vs, w @ vs.abs()
    if gate is not None:
        sg = torch.sigmoid(gate.to(F64))
        out, size = out * sg, size * sg
    return out, size


def norm_rope(x, w, positions, freq, eps, sections=None, interleaved=False, plus_one=True):
    """x [N, heads, D], positions list per axis -> (float64 result, |y_j| + |y_j+R/2| of its pair)."""
    y = x.to(F64)
    if w is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * (w.to(F64) + (1 if plus_one else 0))
    half = len(freq)
    out, size = y.clone(), y.abs()
    axes = len(positions)
    sections = sections or [half]
    owner = []
    for j in range(half):
        if interleaved:
            a = j % axes
            owner.append(a if j < axes * sections[a] else 0)
        else:
            a, left = 0, j
            while left >= sections[a]:
                left -= sections[a]
                a += 1
            owner.append(a)
    for j in range(half):
        for n in range(x.shape[0]):
            z = float(positions[owner[j]][n]) * float(freq[j])
            turned = torch.complex(y[n, :, j], y[n, :, j + half]) * complex(math.cos(z), math.sin(z))
            out[n, :, j], out[n, :, j + half] = turned.real, turned.imag
            size[n, :, j] = size[n, :, j + half] = y[n, :, j].abs() + y[n, :, j + half].abs()
    return out, size
