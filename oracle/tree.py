"""Drafted trees over the caches, in float64, request by request and node by
node: block tables and slots in Python, attention by path, the gated delta rule
and the causal conv token by token along each path."""
from __future__ import annotations

import math

import torch

F64 = torch.float64


def paths(parents, n):
    """For each of a request's n nodes the nodes from the context to it, itself last."""
    out = []
    for i in range(n):
        p = i - 1 if parents is None else int(parents[i])
        out.append((out[p] if 0 <= p < i else []) + [i])
    return out


def _used(x, block, columns, wrap):
    n = -(-max(x, 0) // block)
    return min(n, columns) if wrap else n


def extend(lengths, added, tables, free, count, block, total, wrap=False):
    """Lists (tables, free changed in place) -> (slots, served, count)."""
    columns = len(tables[0])
    slots, served, taken, dry = [], [], 0, False
    for r, (length, a) in enumerate(zip(lengths, added)):
        held, want = _used(length, block, columns, wrap), _used(length + a, block, columns, wrap)
        ok = want <= columns
        need = want - held if ok else 0
        if ok and need:
            dry = dry or taken + need > count
            ok = not dry
        if ok:
            for c in range(held, want):
                tables[r][c] = free[count - 1 - taken]
                taken += 1
        served.append(ok)
        for p in range(length, length + a):   # a ring's row goes to the last of the call that has it
            there = ok and p + columns * block >= length + a
            slots.append(tables[r][p // block % columns] * block + p % block if there else -1)
    return slots + [-1] * (total - len(slots)), served, count - taken


def trim(lengths, kept, tables, free, count, block, wrap=False):
    columns = len(tables[0])
    back = []
    for r, (length, k) in enumerate(zip(lengths, kept)):
        for c in range(_used(k, block, columns, wrap), min(columns, _used(length, block, columns, wrap))):
            if tables[r][c] >= 0:
                back.append(tables[r][c])
                tables[r][c] = -1
    for i, b in enumerate(back):
        free[count + len(back) - 1 - i] = b
    return count + len(back)


def slot_map(cu, lengths, tables, block, total, parents=None, last=None, served=None, wrap=True):
    columns = len(tables[0])
    slots, kept = [-1] * total, []
    for r, length in enumerate(lengths):
        a, n = cu[r], cu[r + 1] - cu[r]
        ps = paths(None if parents is None else parents[a:a + n], n)
        if last is None:
            on, deep = range(n), max((len(x) for x in ps), default=0)
        else:
            on = ps[last[r]] if 0 <= last[r] < n else []
            deep = len(on)
        if (served is not None and not served[r]) or (not wrap and length + deep > columns * block):
            on, deep = [], 0
        kept.append(length + deep)
        for i in on:
            p = length + len(ps[i]) - 1
            if p + columns * block >= kept[-1]:
                slots[a + i] = tables[r][p // block % columns] * block + p % block
    return slots, kept


def attention(q, k, v, parents, cu, lengths, keys, values, tables, window=None, gate=None, scale=None):
    n, h, d = q.shape
    g, block, columns = k.shape[1], keys.shape[2], tables.shape[1]
    scale = d ** -0.5 if scale is None else scale
    out = torch.zeros(n, h, d, dtype=F64)
    for r, length in enumerate(lengths):
        a, b = cu[r], cu[r + 1]
        for i, path in enumerate(paths(None if parents is None else parents[a:b], b - a)):
            pos = length + len(path) - 1
            oldest = max(0, length - columns * block, pos - window + 1 if window else 0)
            at = [p for p in range(oldest, length) if 0 <= int(tables[r, p // block % columns]) < keys.shape[0]]
            ids, rows = [int(tables[r, p // block % columns]) for p in at], [p % block for p in at]
            near = [j for e, j in enumerate(path) if not window or len(path) - 1 - e < window]
            for head in range(h):
                kv = head // (h // g)
                ks = torch.cat((keys[ids, kv, rows], k[[a + j for j in near], kv])).to(F64)
                vs = torch.cat((values[ids, kv, rows], v[[a + j for j in near], kv])).to(F64)
                out[a + i, head] = torch.softmax(ks @ q[a + i, head].to(F64) * scale, 0) @ vs
    return out if gate is None else out * torch.sigmoid(gate.to(F64))


def delta_rule(q, k, v, g, beta, parents, cu, state, rows=None, scale=None, l2=True):
    """[N, heads, dim] inputs -> (o [N, HV, V], the size of its terms: ||q|| scale times the
    norms of the state's columns and of the updates on the path)."""
    q, k, v, g, beta = (x.to(F64) for x in (q, k, v, g, beta))
    if l2:
        q, k = (x / torch.sqrt((x * x).sum(-1, keepdim=True) + 1e-6) for x in (q, k))
    rep, scale = v.shape[1] // q.shape[1], q.shape[2] ** -0.5 if scale is None else scale
    q, k = q.repeat_interleave(rep, 1), k.repeat_interleave(rep, 1)
    out, size = torch.zeros_like(v), torch.zeros_like(v)
    for r in range(len(cu) - 1):
        row = r if rows is None else rows[r]
        if not 0 <= row < state.shape[0]:
            continue
        a, n = cu[r], cu[r + 1] - cu[r]
        for i, path in enumerate(paths(None if parents is None else parents[a:a + n], n)):
            s = state[row].to(F64)
            terms = s.norm(dim=1)
            for j in path:
                j += a
                s = s * torch.exp(g[j])[:, None, None]
                delta = beta[j][:, None] * (v[j] - torch.einsum("hk,hkv->hv", k[j], s))
                s = s + k[j][:, :, None] * delta[:, None]
                terms = terms + k[j].norm(dim=1)[:, None] * delta.abs()
            size[a + i] = q[a + i].norm(dim=1)[:, None] * terms * scale
            out[a + i] = torch.einsum("hk,hkv->hv", q[a + i], s) * scale
    return out, size


def conv(x, window, w, parents, cu):
    """x [N, C], window [R, 3, C], w [C, 4] -> silu(conv) [N, C]."""
    out = torch.zeros(x.shape, dtype=F64)
    for r in range(len(cu) - 1):
        a, n = cu[r], cu[r + 1] - cu[r]
        for i, path in enumerate(paths(None if parents is None else parents[a:a + n], n)):
            taps = torch.cat((window[r], x[[a + j for j in path]])).to(F64)[-4:]
            y = (taps * w.to(F64).T).sum(0)
            out[a + i] = y / (1 + torch.exp(-y))
    return out
