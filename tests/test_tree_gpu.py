"""Drafted trees over the caches on the GPU, against float64 request by request.

Tolerances, from the roundings that each kernel makes (e = half a step of the
output's type, torch.finfo(t).eps / 2):
* attention: the output is rounded once (e |o|) and every weight of the value
  product once (e sum p |v|); scores, exponentials and sums are float32, whose
  error in the exponent (below 2^-24 x 128 terms x the largest score) leaves
  2^-12 sum p |v|.
* delta rule: the output once (e |o|); everything else is float32 or a pair of
  16-bit values (2^-16): 2^-12 of the size of the terms.
* conv: the output once, the four products and the SiLU in float32 (2^-18 of
  the products' size).
* tables, slots and copies are exact.
"""
from dataclasses import fields

import pytest
import torch

from oracle import tree as ref
from yanchor_amd import _native as N
from yanchor_amd import gdn, layers, workloads
from yanchor_amd import independent_memory as im
from yanchor_amd import inference_kernels as ik

pytestmark = pytest.mark.gpu

NAN = float("nan")


def half_step(t):
    return torch.finfo(t).eps / 2


def within(x, want, bound, what=""):
    """|x - want| <= bound everywhere; the worst ratio is told."""
    x = x.detach().double().cpu()
    assert x.shape == want.shape
    bad = (x - want).abs() > bound + 1e-30
    bad |= ~torch.isfinite(x) & torch.isfinite(want)
    ratio = ((x - want).abs() / (bound + 1e-30)).max().item() if x.numel() else 0
    assert not bad.any(), f"{what}: {int(bad.sum())} of {x.numel()} off, {ratio:.2f} times the bound, first at {bad.nonzero()[0].tolist()}"


def trees(counts, seed, back=4):
    """(cu list, parents list) of packed random trees."""
    gen = torch.Generator().manual_seed(seed)
    cu, parents = [0], []
    for n in counts:
        for i in range(n):
            parents.append(max(-1, i - int(torch.randint(1, back + 1, (), generator=gen))))
        cu.append(cu[-1] + n)
    return cu, parents


def rnd(*shape, seed, dtype=torch.bfloat16, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


# --- attention ------------------------------------------------------------------

def attention_case(dev, lengths, counts, *, h=8, g=2, d=128, block=16, columns=None, window=None, gate=None,
                   dtype=torch.bfloat16, chain=False, pad=0, seed=0, max_nodes=None, bad=None, fill=NAN, scale=None,
                   std=1.0, max_length=None):
    cu, parents = trees(counts, seed)
    n = cu[-1]
    if chain:
        parents = None
    columns = columns or max(1, max(-(-x // block) for x in lengths))
    blocks = len(lengths) * columns + 2
    order = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed)).tolist()
    keys, values = (rnd(blocks, g, block, d, seed=seed + s, dtype=dtype) for s in (1, 2))
    tables = torch.full((len(lengths), columns), -1, dtype=torch.int32)
    live = torch.zeros(blocks, block, dtype=torch.bool)
    for r, x in enumerate(lengths):
        for p in range(max(0, x - columns * block), x):
            c = p // block % columns
            tables[r, c] = order[r * columns + c]
            live[tables[r, c], p % block] = True
    dead = ~live[:, None, :, None].expand_as(keys)    # what no position holds may be anything
    keys[dead] = fill
    values[dead] = fill
    for r, c, x in bad or []:
        tables[r, c] = x
    q = rnd(n + pad, h, d, seed=seed + 3, dtype=dtype, std=1.5 * std)
    k, v = (rnd(n + pad, g, d, seed=seed + s, dtype=dtype) for s in (4, 5))
    gt = None
    if gate == "dense":
        gt = rnd(n + pad, h, d, seed=seed + 6, dtype=dtype)
    elif gate == "odd":      # heads interleaved with something else, rows off 8-byte alignment
        gt = rnd(n + pad, h, 2 * d + 1, seed=seed + 6, dtype=dtype)[:, :, d:2 * d]
    for t in (q, k, v):
        t[n:] = NAN
    to = dict(device=dev)
    got = layers.tree_attention(q.to(**to), k.to(**to), v.to(**to), None if parents is None else i32(parents + [7] * pad, dev),
                                i32(cu, dev), torch.tensor(lengths, device=dev), keys.to(**to), values.to(**to),
                                tables.to(**to), window=window, scale=scale, max_nodes=max_nodes, max_length=max_length,
                                gate=None if gt is None else torch.empty_strided(gt.shape, gt.stride(), dtype=dtype, device=dev).copy_(gt))
    args = (parents, cu, lengths, keys)
    want = ref.attention(q[:n], k[:n], v[:n], *args, values, tables, window, None if gt is None else gt[:n], scale)
    size = ref.attention(q[:n], k[:n], v[:n].abs(), *args, values.abs(), tables, window, None, scale)
    if gt is not None:
        size = size * torch.sigmoid(gt[:n].double())
    torch.cuda.synchronize()
    assert torch.equal(got[n:].cpu(), torch.zeros(pad, h, d, dtype=dtype))
    within(got[:n], want, half_step(dtype) * (want.abs() + size) + 2.0 ** -12 * size)
    return got


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float16, 128), (torch.bfloat16, 64),
                                     (torch.float16, 64)])
def test_attention_lengths_and_node_counts(gpu, dtype, d):
    attention_case(gpu, [0, 1, 63, 64, 65, 150, 7, 128], [1, 0, 5, 64, 17, 3, 33, 2], d=d, dtype=dtype, seed=1)


@pytest.mark.parametrize("h,g,block", [(1, 1, 16), (6, 2, 24), (5, 1, 1), (16, 2, 64), (8, 8, 7), (12, 1, 100)])
def test_attention_heads_and_blocks(gpu, h, g, block):
    attention_case(gpu, [70, 5, 131], [9, 64, 1], h=h, g=g, block=block, seed=2)


@pytest.mark.parametrize("window,block,columns", [(40, 40, 1), (64, 64, 1), (1, 16, None), (3, 16, None),
                                                  (100, 16, 8), (50, 24, 3)])
def test_attention_windows_and_rings(gpu, window, block, columns):
    """Rings of one block, rings of blocks, and windows over a whole cache; some not yet full."""
    attention_case(gpu, [0, 39, 40, 41, 300, 1000, 64], [4, 12, 1, 20, 64, 7, 2], window=window, block=block,
                   columns=columns, seed=3)


def test_attention_reads_the_last_positions_that_are_there(gpu):
    attention_case(gpu, [100, 48, 49], [3, 3, 3], block=16, columns=3, seed=4)


@pytest.mark.parametrize("gate", ["dense", "odd"])
def test_attention_gate_padding_and_chains(gpu, gate):
    attention_case(gpu, [33, 90], [6, 11], gate=gate, chain=True, pad=5, seed=5)
    attention_case(gpu, [33, 90], [6, 11], gate=gate, pad=70, seed=6)


def test_attention_of_single_tokens(gpu):
    attention_case(gpu, [513, 0, 1024, 77], [1, 1, 1, 1], chain=True, max_nodes=1, h=32, g=8, seed=7)


def test_attention_long_caches_in_parts(gpu):
    attention_case(gpu, [3000, 70, 900, 4097], [2, 40, 17, 1], h=4, g=2, seed=51)
    attention_case(gpu, [2500, 1300], [64, 3], h=8, g=1, block=64, gate="dense", seed=52)    # 512 rows a head
    attention_case(gpu, [5000], [1], h=2, g=1, d=64, chain=True, max_nodes=1, dtype=torch.float16, seed=53)


def test_attention_of_many_requests(gpu):
    """More requests than a workgroup has threads, some of one token and some of none."""
    gen = torch.Generator().manual_seed(1)
    lengths = torch.randint(0, 90, (700,), generator=gen).tolist()
    lengths[3], lengths[600] = 2000, 1500
    counts = torch.randint(0, 3, (700,), generator=gen).tolist()
    attention_case(gpu, lengths, counts, h=2, g=1, seed=54, window=1200)


@pytest.mark.parametrize("max_length", [None, 10])
def test_attention_of_whole_items(gpu, max_length):
    """So many heads that none is cut; a bound that is too low changes no result."""
    gen = torch.Generator().manual_seed(2)
    lengths = torch.randint(0, 200, (140,), generator=gen).tolist()
    counts = torch.randint(0, 9, (140,), generator=gen).tolist()
    attention_case(gpu, lengths, counts, h=8, g=8, d=64, block=8, window=70, gate="dense", pad=3, seed=55,
                   max_length=max_length, max_nodes=8)
    attention_case(gpu, lengths[:34], [min(64, 8 * x) for x in counts[:34]], h=32, g=8, d=64, block=1, columns=90,
                   seed=56, max_length=max_length)


def test_attention_holes_in_a_table_are_not_seen(gpu):
    attention_case(gpu, [200, 130], [8, 8], bad=[(0, 3, -1), (0, 7, 1 << 30), (1, 0, 10 ** 6), (1, 8, -5)], seed=8)


def test_attention_scale_and_large_scores(gpu):
    """Scores of several hundred: the softmax is nearly one key."""
    attention_case(gpu, [150], [16], scale=1.0, seed=9)
    for scale in (0.0, -1.0, float("inf"), NAN):     # the scores' order is what the masks count on
        with pytest.raises(ValueError, match="positive"):
            attention_case(gpu, [150], [16], scale=scale, seed=10)


def test_attention_equal_keys_and_infinite_keys(gpu):
    """A key of infinities takes all of the weight, or none."""
    dev = gpu
    q = torch.ones(2, 1, 128, dtype=torch.bfloat16, device=dev)
    k = torch.zeros(2, 1, 128, dtype=torch.bfloat16, device=dev)
    v = torch.full((2, 1, 128), 3.0, dtype=torch.bfloat16, device=dev)
    keys = torch.zeros(1, 1, 16, 128, dtype=torch.bfloat16, device=dev)
    values = torch.arange(16, device=dev, dtype=torch.bfloat16)[None, None, :, None].expand(1, 1, 16, 128).contiguous()
    keys[0, 0, 5] = -float("inf")
    out = layers.tree_attention(q, k, v, None, i32([0, 2], dev), torch.tensor([8], device=dev), keys, values,
                                i32([[0]], dev))
    want = torch.tensor([(sum(range(8)) - 5 + 3) / 8, (sum(range(8)) - 5 + 6) / 9], dtype=torch.float64)
    within(out[:, 0, 0], want, want * 2.0 ** -7)


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float16, 64)])
@pytest.mark.parametrize("value", [NAN, float("inf")])
def test_attention_keeps_what_is_not_finite_on_its_path(gpu, dtype, d, value):
    """A node's key or value reaches its descendants, a cached one the nodes whose window holds it."""
    cu, parents = trees([40, 20], 61)
    n, lengths, window = cu[-1], [130, 90], 70
    q, k, v = rnd(n, 8, d, seed=1, dtype=dtype), rnd(n, 2, d, seed=2, dtype=dtype), rnd(n, 2, d, seed=3, dtype=dtype)
    keys, values = (rnd(20, 2, 16, d, seed=s, dtype=dtype) for s in (4, 5))
    tables = torch.arange(20, dtype=torch.int32).view(2, 10)
    call = lambda k, v, values: layers.tree_attention(  # noqa: E731
        q.to(gpu), k.to(gpu), v.to(gpu), i32(parents, gpu), i32(cu, gpu), torch.tensor(lengths, device=gpu), keys.to(gpu),
        values.to(gpu), tables.to(gpu), window=window).cpu()
    args = (parents, cu, lengths, keys)
    want = ref.attention(q, k, v, *args, values, tables, window)
    size = ref.attention(q, k, v.abs(), *args, values.abs(), tables, window)
    bound = half_step(dtype) * (want.abs() + size) + 2.0 ** -12 * size
    p = 62                                       # request 0's position, at the edge of its nodes' windows
    for which in ("k", "v", "cache"):
        k2, v2, c2 = k.clone(), v.clone(), values.clone()
        if which == "cache":
            c2[tables[0, p // 16], :, p % 16, 3] = value
        else:
            (k2 if which == "k" else v2)[7, :, 3] = value
            (k2 if which == "k" else v2)[45, :, 3] = value
        got = call(k2, v2, c2)
        for r in range(2):
            for i, path in enumerate(ref.paths(parents[cu[r]:cu[r + 1]], cu[r + 1] - cu[r])):
                row = cu[r] + i
                if which == "cache":
                    sees = r == 0 and lengths[0] + len(path) - 1 - p < window
                else:
                    sees = 7 - cu[r] in path or 45 - cu[r] in path
                if sees and which != "k":
                    assert not torch.isfinite(got[row, :, 3]).any(), (which, row)
                elif not sees:
                    within(got[row], want[row], bound[row], (which, row))


def test_attention_counts_past_max_nodes(gpu):
    """Nodes past the most are not-a-number, the others as ever."""
    q, k, v = (rnd(80, 2, 64, seed=s).to(gpu) for s in (1, 2, 3))
    cache = rnd(1, 2, 16, 64, seed=4).to(gpu)
    args = (torch.tensor([5, 9], device=gpu), cache, cache, i32([[0], [0]], gpu))
    out = layers.tree_attention(q, k, v, None, i32([0, 70, 80], gpu), *args)
    assert out[64:70].isnan().all() and not out[:64].isnan().any() and not out[70:].isnan().any()
    few = layers.tree_attention(q, k, v, None, i32([0, 70, 80], gpu), *args, max_nodes=8)
    assert torch.equal(few[:8], out[:8]) and few[8:70].isnan().all() and torch.equal(few[70:78], out[70:78])


def test_attention_empty_calls(gpu):
    z = torch.zeros(0, 4, 64, dtype=torch.bfloat16, device=gpu)
    cache = torch.zeros(0, 4, 16, 64, dtype=torch.bfloat16, device=gpu)
    none = torch.zeros(0, dtype=torch.int64, device=gpu)
    out = layers.tree_attention(z, z, z, None, i32([0], gpu), none, cache, cache, torch.zeros(0, 1, dtype=torch.int32, device=gpu))
    assert out.shape == (0, 4, 64)
    three = torch.ones(3, 4, 64, dtype=torch.bfloat16, device=gpu)   # rows, but no request
    out = layers.tree_attention(three, three, three, None, i32([0], gpu), none, cache, cache,
                                torch.zeros(0, 1, dtype=torch.int32, device=gpu))
    assert torch.equal(out, torch.zeros_like(three))


def test_attention_at_the_last_positions(gpu):
    """Rings at positions near 2^31 read as at the same rows of early positions."""
    cu, parents = trees([9, 64], 5)
    q = rnd(cu[-1], 8, 128, seed=1).to(gpu)
    k, v = (rnd(cu[-1], 2, 128, seed=s).to(gpu) for s in (2, 3))
    keys, values = (rnd(2, 2, 1024, 128, seed=s).to(gpu) for s in (4, 5))
    tables, par, off = i32([[1], [0]], gpu), i32(parents, gpu), i32(cu, gpu)
    late = torch.tensor([2 ** 31 - 4096, 2 ** 31 - 5000], device=gpu)
    runs = [layers.tree_attention(q, k, v, par, off, x, keys, values, tables, window=1024)
            for x in (late, late - 1024 * (2 ** 21 - 16))]
    assert torch.equal(*runs) and torch.isfinite(runs[0]).all()


def test_caches_past_32_bit_offsets(gpu):
    """Blocks, state rows and slots whose offsets pass 2^31 elements, against a small cache with the same rows."""
    g, block, d, few = 8, 64, 128, 6
    blocks = 2 ** 31 // (g * block * d) + few
    big = [torch.empty(blocks, g, block, d, dtype=torch.bfloat16, device=gpu) for _ in range(2)]
    small = [torch.empty(few, g, block, d, dtype=torch.bfloat16, device=gpu) for _ in range(2)]
    k, v = (rnd(few * block, g, d, seed=s).to(gpu) for s in (1, 2))
    slots = torch.arange(few * block, device=gpu)
    layers.cache_write(k, v, slots + (blocks - few) * block, *big)
    layers.cache_write(k, v, slots, *small)
    assert torch.equal(big[0][-few:], small[0]) and torch.equal(big[1][-few:], small[1])
    cu, parents = trees([7, 20], 3)
    q = rnd(cu[-1], 32, d, seed=3).to(gpu)
    tables = torch.tensor([[4, 0, 2], [5, 1, 3]], dtype=torch.int32, device=gpu)
    args = (q, k[:cu[-1]], v[:cu[-1]], i32(parents, gpu), i32(cu, gpu), torch.tensor([130, 192], device=gpu))
    assert torch.equal(layers.tree_attention(*args, *big, tables + (blocks - few)),
                       layers.tree_attention(*args, *small, tables))
    del big
    rows = 2 ** 31 // (32 * 128 * 128) + 2
    pool = torch.empty(rows, 32, 128, 128, device=gpu)
    state = rnd(2, 32, 128, 128, seed=4, dtype=torch.float32).to(gpu)
    pool[-2:] = state
    qk = [rnd(1, cu[-1], 32, 128, seed=s).to(gpu) for s in (5, 6, 7)]
    gb = [-torch.rand(1, cu[-1], 32, device=gpu), torch.rand(1, cu[-1], 32, device=gpu)]
    for x in (qk, [t.float() for t in qk]):
        assert torch.equal(gdn.tree_gated_delta_rule(*x, *gb, *args[3:5], pool, state_indices=i32([rows - 1, rows - 2], gpu)),
                           gdn.tree_gated_delta_rule(*x, *gb, *args[3:5], state, state_indices=i32([1, 0], gpu)))


# --- gated delta rule -------------------------------------------------------------

def delta_case(dev, counts, *, h=2, hv=4, kd=128, vd=128, dtype=torch.bfloat16, state=torch.float32, rows=None, pad=0,
               l2=True, scale=None, gates=(torch.float32, torch.float32), chain=False, seed=0, max_nodes=None,
               decay=1.0):
    cu, parents = trees(counts, seed)
    if chain:
        parents = None
    n = cu[-1]
    pool = len(counts) + 2
    q, k = (rnd(1, n + pad, h, kd, seed=seed + s, dtype=dtype, std=1.0 if l2 else kd ** -0.5) for s in (1, 2))
    v = rnd(1, n + pad, hv, vd, seed=seed + 3, dtype=dtype)
    g = (-decay * torch.rand(1, n + pad, hv, generator=torch.Generator().manual_seed(seed + 4))).to(gates[0])
    beta = torch.sigmoid(rnd(1, n + pad, hv, seed=seed + 5, dtype=torch.float32)).to(gates[1])
    s0 = rnd(pool, hv, kd, vd, seed=seed + 6, dtype=state, std=0.3)
    for t in (q, k, v, g, beta):
        t[:, n:] = NAN
    on = [x.to(dev) for x in (q, k, v, g, beta)]
    got = gdn.tree_gated_delta_rule(*on, None if parents is None else i32(parents + [3] * pad, dev), i32(cu, dev), s0.to(dev),
                                    state_indices=None if rows is None else i32(rows, dev), scale=scale,
                                    use_qk_l2norm_in_kernel=l2, max_nodes=max_nodes)
    want, size = ref.delta_rule(q[0, :n], k[0, :n], v[0, :n], g[0, :n], beta[0, :n], parents, cu, s0, rows, scale, l2)
    torch.cuda.synchronize()
    assert torch.equal(got[0, n:].cpu(), torch.zeros(pad, hv, vd, dtype=dtype))
    within(got[0, :n], want, half_step(dtype) * want.abs() + 2.0 ** -12 * size)


@pytest.mark.parametrize("vd,state", [(128, torch.float32), (64, torch.float32), (128, torch.float16),
                                      (64, torch.float16)])
def test_delta_rule_node_counts(gpu, vd, state):
    delta_case(gpu, [1, 0, 5, 16, 17, 33, 48, 64, 63], vd=vd, state=state, seed=11)


@pytest.mark.parametrize("counts,most", [([1, 1, 1], 1), ([7, 2], 7), ([16, 3], 16), ([17, 1], 17), ([32, 9], 32)])
def test_delta_rule_small_trees(gpu, counts, most):
    delta_case(gpu, counts, max_nodes=most, seed=12)


@pytest.mark.parametrize("kd,vd,dtype", [(64, 64, torch.bfloat16), (64, 128, torch.float32), (128, 128, torch.float16),
                                         (128, 64, torch.float32)])
def test_delta_rule_other_types(gpu, kd, vd, dtype):
    delta_case(gpu, [3, 20, 64], kd=kd, vd=vd, dtype=dtype, gates=(dtype, torch.float32), seed=13)


def test_delta_rule_rows_padding_and_options(gpu):
    delta_case(gpu, [4, 9, 2, 6], rows=[5, -1, 0, 3], pad=6, seed=14)
    delta_case(gpu, [4, 9], rows=[1, 1], pad=70, chain=True, seed=15)          # one state, two drafts
    delta_case(gpu, [20, 9], l2=False, scale=0.7, h=4, gates=(torch.bfloat16, torch.float16), seed=16)
    delta_case(gpu, [30, 64], decay=40.0, seed=17)     # decays that underflow along a path
    delta_case(gpu, [30, 64], decay=0.0, chain=True, seed=18)


def test_delta_rule_counts_past_max_nodes(gpu):
    x, v = rnd(1, 80, 2, 128, seed=1).to(gpu), rnd(1, 80, 2, 128, seed=2).to(gpu)
    g, b, s = torch.zeros(1, 80, 2, device=gpu), torch.ones(1, 80, 2, device=gpu), torch.zeros(2, 2, 128, 128, device=gpu)
    o = gdn.tree_gated_delta_rule(x, x, v, g, b, None, i32([0, 70, 80], gpu), s)
    assert o[0, 64:70].isnan().all() and not o[0, :64].isnan().any() and not o[0, 70:].isnan().any()


@pytest.mark.parametrize("which", ["q", "k", "v", "g", "beta"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_delta_rule_keeps_what_is_not_finite_on_its_path(gpu, which, dtype):
    cu, parents = trees([40, 20], 41)
    n = cu[-1]
    x = dict(q=rnd(1, n, 2, 128, seed=1, dtype=dtype), k=rnd(1, n, 2, 128, seed=2, dtype=dtype),
             v=rnd(1, n, 2, 128, seed=3, dtype=dtype), g=-torch.rand(1, n, 2), beta=torch.rand(1, n, 2))
    s0 = rnd(2, 2, 128, 128, seed=4, dtype=torch.float32)
    call = lambda: gdn.tree_gated_delta_rule(*(x[t].to(gpu) for t in ("q", "k", "v", "g", "beta")), i32(parents, gpu),  # noqa: E731
                                             i32(cu, gpu), s0.to(gpu))[0].cpu()
    clean = call()
    for at, value in ((7, NAN), (45, float("inf"))):
        x[which][0, at] = value
    got = call()
    for r in range(2):
        for i, path in enumerate(ref.paths(parents[cu[r]:cu[r + 1]], cu[r + 1] - cu[r])):
            row = cu[r] + i
            if 7 - cu[r] in path or 45 - cu[r] in path:
                if which != "q" or row in (7, 45):     # a query is its own node's alone
                    assert not torch.isfinite(got[row]).all()
                    continue
            assert torch.equal(got[row], clean[row]), row


# --- conv ------------------------------------------------------------------------

@pytest.mark.parametrize("channels,planes,extra,chain", [(24, 3, 8, False), (4096, 1, 0, False), (30, 3, 1, False),
                                                         (6144, 3, 4160, True), (9, 1, 2, True)])
def test_conv(gpu, channels, planes, extra, chain):
    counts = [1, 0, 2, 3, 64, 17]
    cu, parents = trees(counts, 21)
    n, pad = cu[-1], 3
    proj = rnd(n + pad, channels + extra, seed=22)
    window, w = rnd(len(counts), 3, channels, seed=23), rnd(channels, 4, seed=24, std=0.5)
    got = layers.conv_tree(proj.to(gpu), window.to(gpu), w.to(gpu), None if chain else i32(parents + [0] * pad, gpu), i32(cu, gpu),
                           channels, planes=planes)
    if planes > 1:
        got = got.transpose(0, 1).reshape(n + pad, channels)
    x = proj[:n, :channels]
    want = ref.conv(x, window, w, None if chain else parents, cu)
    one = torch.ones(1, dtype=torch.float64)
    a = torch.zeros_like(want)
    for r in range(len(counts)):   # the size of the four products
        for i, path in enumerate(ref.paths(None if chain else parents[cu[r]:cu[r + 1]], counts[r])):
            taps = torch.cat((window[r], x[[cu[r] + j for j in path]])).double()[-4:]
            a[cu[r] + i] = (taps * w.double().T).abs().sum(0) * one
    assert not got[n:].any()
    within(got[:n], want, 2.0 ** -8 * want.abs() + 2.0 ** -18 * a)


# --- tables, slots, write -----------------------------------------------------------

@pytest.mark.parametrize("n,block,columns,wrap,most", [(1, 16, 4, False, 20), (5, 16, 5, False, 30), (40, 1, 60, False, 20),
                                                       (300, 7, 8, True, 60), (1500, 16, 9, False, 60),
                                                       (70, 64, 1000, False, 3000)])
def test_extend_and_trim(gpu, n, block, columns, wrap, most):
    gen = torch.Generator().manual_seed(n)
    lengths = torch.randint(0, most, (n,), generator=gen).tolist()
    added = torch.randint(0, most, (n,), generator=gen).tolist()
    pad = 9
    for share in (1.0, 0.4):      # enough blocks, and a stack that runs dry
        tables = [[-1] * columns for _ in range(n)]
        big = list(range(10 ** 6, 10 ** 6 + sum(ref._used(x, block, columns, wrap) for x in lengths)))
        ok = ref.extend([0] * n, lengths, tables, big, len(big), block, sum(lengths), wrap)[1]
        need = sum(ref._used(a + b, block, columns, wrap) - ref._used(a, block, columns, wrap)
                   for a, b in zip(lengths, added))
        free = torch.randperm(int(need * share) + 3, generator=gen).tolist() + [-1] * 5
        count = len(free) - 5
        cu = torch.tensor([0] + added).cumsum(0)
        total = int(cu[-1]) + pad
        t_dev, f_dev = i32(tables, gpu), i32(free, gpu)
        c_dev = i32([count], gpu)
        start = (t_dev.clone(), f_dev[:count].clone())
        slots, served = ik.extend_block_tables(torch.tensor(lengths, device=gpu), cu.to(gpu), t_dev, f_dev, c_dev, block,
                                               total, wrap=wrap)
        want, serve, left = ref.extend(lengths, added, tables, free, count, block, total, wrap)
        assert served.tolist() == serve and slots.tolist() == want
        assert c_dev.tolist() == [left] and t_dev.tolist() == tables
        longer = [a + b for a, b in zip(lengths, added)]
        ik.trim_block_tables(torch.tensor(longer, device=gpu), torch.tensor(lengths, device=gpu), t_dev, f_dev, c_dev, block,
                             wrap=wrap)
        assert ref.trim(longer, lengths, tables, free, left, block, wrap) == c_dev.item() == count
        assert torch.equal(t_dev, start[0]) and torch.equal(f_dev[:count], start[1])
        assert all(ok) or not wrap
        ik.trim_block_tables(torch.tensor(lengths, device=gpu), torch.zeros(n, dtype=torch.int64, device=gpu), t_dev, f_dev,
                             c_dev, block, wrap=wrap)
        assert (t_dev == -1).all()       # the stack may be too small for them all; nothing is written behind it


@pytest.mark.parametrize("n,block,columns", [(3, 4, 2), (1, 1, 1), (40, 16, 3), (1030, 8, 2)])
def test_a_ring_takes_more_tokens_than_it_holds(gpu, n, block, columns):
    """Of the tokens that share a row the last is written, in one launch and in several."""
    gen = torch.Generator().manual_seed(n)
    room = block * columns
    lengths = torch.randint(0, 3 * room, (n,), generator=gen).tolist()
    added = torch.randint(0, 4 * room, (n,), generator=gen).tolist()
    tables = torch.randperm(n * columns, generator=gen).view(n, columns).to(torch.int32).tolist()
    for r, x in enumerate(lengths):
        tables[r][ref._used(x, block, columns, True):] = [-1] * (columns - ref._used(x, block, columns, True))
    free = [x for x in range(n * columns) if x not in {y for t in tables for y in t}]
    cu = torch.tensor([0] + added).cumsum(0)
    total = int(cu[-1])
    t_dev, f_dev, c_dev = i32(tables, gpu), i32(free + [-1], gpu), i32([len(free)], gpu)
    len_dev = torch.tensor(lengths, device=gpu)
    slots, served = ik.extend_block_tables(len_dev, cu.to(gpu), t_dev, f_dev, c_dev, block, total, wrap=True)
    want, serve, _ = ref.extend(lengths, added, tables, free, len(free), block, total, True)
    assert served.tolist() == serve == [True] * n and slots.tolist() == want and t_dev.tolist() == tables
    again, kept = ik.slot_map(cu.to(gpu), len_dev, t_dev, block, total)
    assert torch.equal(again, slots) and kept.tolist() == [a + b for a, b in zip(lengths, added)]
    last = [min(room, x) - 1 for x in added]           # a part of each chain
    got, _ = ik.slot_map(cu.to(gpu), len_dev, t_dev, block, total, last=i32(last, gpu))
    assert got.tolist() == ref.slot_map(cu.tolist(), lengths, tables, block, total, last=last)[0]
    short = [min(x, 64) for x in added]                # as trees
    par, off = [i - 1 for x in short for i in range(x)], torch.tensor([0] + short).cumsum(0)
    got, _ = ik.slot_map(off.to(gpu), len_dev, t_dev, block, len(par), parents=i32(par, gpu))
    assert got.tolist() == ref.slot_map(off.tolist(), lengths, tables, block, len(par), par)[0]
    k = torch.arange(total, device=gpu, dtype=torch.float32).view(-1, 1, 1).expand(total, 2, 4).contiguous()
    keys = torch.full((n * columns, 2, block, 4), -1.0, device=gpu)
    values = keys.clone()
    layers.cache_write(k, -k, slots, keys, values)
    exact = torch.full((n * columns, block), -1.0)
    for r in range(n):                                 # one after the other
        for i in range(added[r]):
            p = lengths[r] + i
            exact[tables[r][p // block % columns], p % block] = float(cu[r] + i)
    assert torch.equal(keys.cpu(), exact[:, None, :, None].expand_as(keys))
    assert torch.equal(values.cpu(), torch.where(exact < 0, exact, -exact)[:, None, :, None].expand_as(keys))


@pytest.mark.parametrize("tree", [True, False])
def test_slot_map(gpu, tree):
    counts = [5, 0, 64, 1, 17] if tree else [5, 0, 200, 1, 17]
    cu, parents = trees(counts, 31)
    lengths, block, columns = [3, 8, 100, 0, 61], 16, 21
    tables = torch.randperm(len(counts) * columns, generator=torch.Generator().manual_seed(1)).view(-1, columns).to(torch.int32)
    tables[4, 4] = -1           # position 64 on: not served
    par = parents if tree else None
    pad = 6
    args = (i32(cu, gpu), torch.tensor(lengths, device=gpu), tables.to(gpu), block, cu[-1] + pad)
    dev_par = None if par is None else i32(par + [0] * pad, gpu)
    for last in (None, [4, -1, 40, 0, 16], [-1, 0, 63, 5, 3]):
        slots, kept = ik.slot_map(*args, parents=dev_par, last=None if last is None else i32(last, gpu))
        got, want = slots.tolist(), ref.slot_map(cu, lengths, tables.tolist(), block, cu[-1] + pad, par,
                                                 None if last is None else [min(x, c - 1) if not tree else x for x, c in zip(last, counts)])
        assert kept.tolist() == want[1]
        assert got == [-1 if x < 0 else x for x in want[0]]


@pytest.mark.parametrize("dtype,g,d,block", [(torch.bfloat16, 8, 128, 16), (torch.float16, 5, 64, 1),
                                             (torch.float32, 3, 12, 7), (torch.bfloat16, 1, 8, 1024)])
def test_cache_write(gpu, dtype, g, d, block):
    for n in (1, 3, 300):
        blocks = -(-n // block) + 2
        gen = torch.Generator().manual_seed(n)
        slots = torch.randperm(blocks * block, generator=gen)[:n]
        slots[torch.rand(n, generator=gen) < 0.3] = -1
        if n > 1:
            slots[0] = blocks * block     # past the cache
        wide = rnd(n, 3 * g * d, seed=n, dtype=dtype)
        k, v = wide[:, :g * d].view(n, g, d), wide[:, 2 * g * d:].view(n, g, d)
        keys, values = (torch.full((blocks, g, block, d), NAN, dtype=dtype) for _ in range(2))
        pos, cpos = torch.arange(n) + 7, torch.full((blocks, g, block), -1, dtype=torch.int32)
        dk, dv, dp = keys.to(gpu), values.to(gpu), cpos.to(gpu)
        w = wide.to(gpu)
        layers.cache_write(w[:, :g * d].view(n, g, d), w[:, 2 * g * d:].view(n, g, d), slots.to(gpu), dk, dv,
                           positions=pos.to(gpu), cache_positions=dp)
        for i, s in enumerate(slots.tolist()):
            if 0 <= s < blocks * block:
                keys[s // block, :, s % block], values[s // block, :, s % block] = k[i], v[i]
                cpos[s // block, :, s % block] = pos[i]
        assert torch.equal(dk.cpu().nan_to_num(9.5), keys.nan_to_num(9.5))
        assert torch.equal(dv.cpu().nan_to_num(9.5), values.nan_to_num(9.5)) and torch.equal(dp.cpu(), cpos)


# --- odd arguments, streams, graphs, and the operators together -------------------------

def test_odd_parents_and_offsets(gpu):
    """A parent that is not an earlier node is the context; offsets past the rows are clamped."""
    n = 9
    q, k, v = rnd(n, 4, 64, seed=1).to(gpu), rnd(n, 2, 64, seed=2).to(gpu), rnd(n, 2, 64, seed=3).to(gpu)
    cache, tables = rnd(4, 2, 16, 64, seed=4).to(gpu), i32([[0, 1], [2, 3]], gpu)
    lens = torch.tensor([20, 30], device=gpu)
    call = lambda parents, cu: layers.tree_attention(q, k, v, parents, cu, lens, cache, cache, tables)  # noqa: E731
    plain = call(i32([-1, 0, -1, -1, -1, 0, -1, -1, 2], gpu), i32([0, 5, 9], gpu))
    odd = call(i32([7, 0, 2, -9, 2 ** 31 - 1, 0, 1, 2, 2], gpu), i32([0, 5, 9], gpu))
    assert torch.equal(plain, odd)
    assert torch.equal(plain, call(torch.tensor([-1, 0, -1, -1, -1, 0, -1, -1, 2]), torch.tensor([0, 5, 9])))  # int64, from the host
    wild = call(None, i32([-3, 5, 4000], gpu))
    assert torch.equal(wild, call(None, i32([0, 5, 9], gpu)))
    x, w = rnd(1, n, 2, 128, seed=5).to(gpu), rnd(2, 3, 48, seed=6).to(gpu)
    gates, state = torch.rand(1, n, 2, device=gpu), torch.rand(2, 2, 128, 128, device=gpu)
    for cu in ([-3, 5, 4000], [0, 7, 3]):
        gdn.tree_gated_delta_rule(x, x, x, -gates, gates, None, i32(cu, gpu), state)
        layers.conv_tree(rnd(n, 48, seed=7).to(gpu), w, rnd(48, 4, seed=8).to(gpu), None, i32(cu, gpu), 48)
        ik.slot_map(i32(cu, gpu), lens, tables, 16, n, parents=i32([0] * n, gpu))
        ik.slot_map(i32(cu, gpu), lens, tables, 16, n)
        free = torch.arange(6, dtype=torch.int32, device=gpu)
        slots, _ = ik.extend_block_tables(lens, i32(cu, gpu), tables.clone(), free, i32([99], gpu), 16, n)
    torch.cuda.synchronize()


def test_strided_rows_and_broadcast_inputs(gpu):
    """Columns of wider projections, single rows, expanded tensors: as their copies."""
    wide = rnd(6, 5 * 128, seed=1).to(gpu)
    q, k, v = wide[:, :256].view(6, 2, 128), wide[:, 256:384].view(6, 1, 128), wide[:, 512:].view(6, 1, 128)
    cache = rnd(3, 1, 16, 128, seed=2).to(gpu)
    args = (None, i32([0, 6], gpu), torch.tensor([40], device=gpu), cache, cache, i32([[2, 0, 1]], gpu))
    assert torch.equal(layers.tree_attention(q, k, v, *args), layers.tree_attention(q.contiguous(), k.contiguous(), v.contiguous(), *args))
    kx = k[:1].expand(6, 1, 128)
    assert torch.equal(layers.tree_attention(q, kx, v, *args), layers.tree_attention(q, kx.contiguous(), v, *args))
    odd = rnd(6, 385, seed=3).to(gpu)[:, 1:257].view(6, 2, 128)       # rows off 16-byte alignment
    gate = rnd(2, 6, 128, seed=4).to(gpu).transpose(0, 1)            # heads outermost
    assert torch.equal(layers.tree_attention(odd, k, v, *args, gate=gate),
                       layers.tree_attention(odd.clone(memory_format=torch.contiguous_format), k, v, *args, gate=gate.contiguous()))
    one = tuple(x[3:4] for x in (q, k, v))
    single = (None, i32([0, 1], gpu), *args[2:])
    assert torch.equal(layers.tree_attention(*one, *single), layers.tree_attention(*(x.clone() for x in one), *single))
    proj = rnd(6, 49, seed=5).to(gpu)
    win, w = rnd(1, 3, 24, seed=6).to(gpu), rnd(24, 4, seed=7).to(gpu)
    assert torch.equal(layers.conv_tree(proj, win, w, *args[:2], 24), layers.conv_tree(proj[:, :24].contiguous(), win, w, *args[:2], 24))


def _step(gpu, seed):
    """What a speculative step holds: the trees, the caches, the states."""
    counts = [7, 1, 20, 0, 12]
    cu, parents = trees(counts, seed)
    n, lengths, block, columns = cu[-1], [50, 3, 161, 90, 16], 16, 14
    gen = torch.Generator().manual_seed(seed)
    tables = torch.full((5, columns), -1, dtype=torch.int32)
    order = torch.randperm(60, generator=gen).to(torch.int32)
    at = 0
    for r, x in enumerate(lengths):
        m = -(-x // block)
        tables[r, :m] = order[at:at + m]
        at += m
    free = torch.cat((order[at:], torch.full((at,), -1, dtype=torch.int32)))
    d = dict(cu=i32(cu, gpu), parents=i32(parents, gpu), lengths=torch.tensor(lengths, device=gpu), tables=tables.to(gpu),
             free=free.to(gpu), count=i32([60 - at], gpu), keys=rnd(60, 2, block, 128, seed=seed).to(gpu),
             values=rnd(60, 2, block, 128, seed=seed + 1).to(gpu), q=rnd(n, 4, 128, seed=seed + 2).to(gpu),
             k=rnd(n, 2, 128, seed=seed + 3).to(gpu), v=rnd(n, 2, 128, seed=seed + 4).to(gpu),
             proj=rnd(n, 3 * 512, seed=seed + 5).to(gpu), window=rnd(5, 3, 3 * 512, seed=seed + 6).to(gpu),
             conv_w=rnd(3 * 512, 4, seed=seed + 7, std=0.5).to(gpu), g=-torch.rand(1, n, 4, generator=gen).to(gpu),
             beta=torch.rand(1, n, 4, generator=gen).to(gpu), state=rnd(5, 4, 128, 128, seed=seed + 8, dtype=torch.float32).to(gpu),
             last=i32([4, -1, 13, -1, 0], gpu))
    return d, cu, parents, lengths, block


def _run_step(s, block):
    n = s["q"].shape[0]
    slots, served = ik.extend_block_tables(s["lengths"], s["cu"], s["tables"], s["free"], s["count"], block, n)
    read = layers.tree_attention(s["q"], s["k"], s["v"], s["parents"], s["cu"], s["lengths"], s["keys"], s["values"], s["tables"])
    x = layers.conv_tree(s["proj"], s["window"], s["conv_w"], s["parents"], s["cu"], 3 * 512, planes=3).view(3, 1, n, 4, 128)
    o = gdn.tree_gated_delta_rule(x[0], x[1], x[2], s["g"], s["beta"], s["parents"], s["cu"], s["state"])
    at, kept = ik.slot_map(s["cu"], s["lengths"], s["tables"], block, n, parents=s["parents"], last=s["last"])
    layers.cache_write(s["k"], s["v"], at, s["keys"], s["values"])
    longer = s["lengths"] + (s["cu"][1:] - s["cu"][:-1])
    ik.trim_block_tables(longer, kept, s["tables"], s["free"], s["count"], block)
    return slots, served, read, x, o, at, kept


def test_a_verification_step(gpu):
    """The operators in one step, against the decode operators run along every path, and the caches that
    the accepted paths leave against the ones that decoding them would."""
    s, cu, parents, lengths, block = _step(gpu, 71)
    before = {k: v.clone() for k, v in s.items()}
    slots, served, read, x, o, at, kept = _run_step(s, block)
    assert served.all()
    vmax, window = 8.0, 256                     # a ring that holds every context whole
    size = []
    for r, length in enumerate(lengths):
        ids = before["tables"][r].cpu().tolist()
        ring = [torch.zeros(1, 2, window, 128, dtype=torch.bfloat16, device=gpu) for _ in range(2)]
        pos = torch.full((1, 2, window), -1, dtype=torch.int32, device=gpu)
        for p in range(length):
            for c, name in zip(ring, ("keys", "values")):
                c[0, :, p] = before[name][ids[p // block], :, p % block]
        pos[0, :, :length] = torch.arange(length, dtype=torch.int32, device=gpu)
        for i, path in enumerate(ref.paths(parents[cu[r]:cu[r + 1]], cu[r + 1] - cu[r])):
            rows = torch.tensor([cu[r] + j for j in path], device=gpu)
            m = len(path)
            rk, rv, rp = ring[0].clone(), ring[1].clone(), pos.clone()
            layers.ring_fill(s["k"][rows], s["v"][rows], i32([0, m], gpu), torch.tensor([length], device=gpu),
                             torch.tensor([0], device=gpu), rk, rv, rp)
            seq = im.ring_decode_attention(s["q"][rows[-1]][None, None], rk, rv, rp)[0, 0].double().cpu()
            within(read[rows[-1]], seq, 2 * (2.0 ** -8 + 2.0 ** -12) * (seq.abs() + vmax), ("attention", r, i))
            win = s["window"][r:r + 1].clone()
            conv = layers.conv_prefill(s["proj"][rows].contiguous(), win, s["conv_w"], i32([0, m], gpu), 3 * 512, planes=3)
            mine = x[:, 0, rows].reshape(3, m, 512).double().cpu()
            within(mine, conv.double().cpu(), 2.0 ** -7 * conv.double().cpu().abs() + 2.0 ** -14, ("conv", r, i))
            y = x[:, :, rows]
            seq, _ = gdn.recurrent_gated_delta_rule(y[0], y[1], y[2], g=s["g"][:, rows], beta=s["beta"][:, rows],
                                                    initial_state=s["state"][r:r + 1].clone())
            _, terms = ref.delta_rule(*(t[0].cpu() for t in (y[0], y[1], y[2], s["g"][:, rows], s["beta"][:, rows])), None,
                                      [0, m], s["state"][r:r + 1].cpu())
            seq = seq[0, -1].double().cpu()
            within(o[0, rows[-1]], seq, 2 * (2.0 ** -8 * seq.abs() + 2.0 ** -12 * terms[-1]), ("delta", r, i))
            size.append(m)
        last = int(s["last"][r])
        path = ref.paths(parents[cu[r]:cu[r + 1]], cu[r + 1] - cu[r])[last] if last >= 0 else []
        assert int(kept[r]) == length + len(path)
        now = s["tables"][r].cpu().tolist()
        for p in range(length + len(path)):         # the cache that decoding the accepted path would leave
            row = s["keys"][now[p // block], :, p % block]
            want = before["keys"][ids[p // block], :, p % block] if p < length else s["k"][cu[r] + path[p - length]]
            assert torch.equal(row, want), (r, p)
        assert now[-(-(length + len(path)) // block):] == [-1] * (len(now) + -(length + len(path)) // block)
    assert max(size) > 3
    used = sum(-(-int(x) // block) for x in kept)
    assert int(s["count"]) == 60 - used
    held = s["tables"][s["tables"] >= 0].tolist() + s["free"][:60 - used].tolist()
    assert sorted(held) == list(range(60))


def test_a_captured_step_replays(gpu):
    """The whole step in a graph, replayed with other inputs and eager work between, against eager runs."""
    s, _, _, _, block = _step(gpu, 81)
    start = {k: v.clone() for k, v in s.items()}

    def reset(seed):
        for k in s:
            s[k].copy_(start[k])
        for j, k in enumerate(("q", "k", "v", "proj")):
            s[k].copy_(rnd(*s[k].shape, seed=seed + j))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _run_step(s, block)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    reset(0)
    with torch.cuda.graph(graph):
        out = _run_step(s, block)
    for seed in (100, 200, 300, 100):
        reset(seed)
        want = [t.clone() for t in _run_step(s, block)]
        after = {k: v.clone() for k, v in s.items()}
        reset(seed)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)
        for k in s:
            assert torch.equal(s[k], after[k]), k


def test_calls_on_two_streams(gpu):
    """Two long calls that overlap, each with scratch of its own."""
    cache = rnd(200, 2, 64, 128, seed=1).to(gpu)
    tables = torch.arange(200, dtype=torch.int32, device=gpu).view(2, 100)
    lens = torch.tensor([6000, 5100], device=gpu)
    ins = [[rnd(24, h, 128, seed=s + i).to(gpu) for i, h in enumerate((8, 2, 2))] for s in (10, 20)]
    call = lambda x: layers.tree_attention(*x, None, i32([0, 11, 24], gpu), lens, cache, cache, tables)  # noqa: E731
    want = [call(x) for x in ins]
    streams = [torch.cuda.Stream() for _ in ins]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for x, st in zip(ins, streams):
            with torch.cuda.stream(st):
                got.append(call(x))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_the_same_bits_every_time(gpu):
    cache = rnd(400, 2, 16, 128, seed=1).to(gpu)
    tables = torch.arange(400, dtype=torch.int32, device=gpu).view(2, 200)
    x = [rnd(70, h, 128, seed=i).to(gpu) for i, h in enumerate((16, 2, 2))]
    call = lambda: layers.tree_attention(*x, None, i32([0, 64, 70], gpu), torch.tensor([3100, 2000], device=gpu), cache, cache, tables)  # noqa: E731
    want = call()
    assert all(torch.equal(call(), want) for _ in range(5))


@pytest.mark.parametrize("tree", [True, False])
@pytest.mark.parametrize("requests,columns,blocks", [(9, 6, 40), (12, 3, 200), (40, 7, 170), (1100, 5, 3600)])
def test_a_step_that_refuses_requests(gpu, tree, requests, columns, blocks):
    """Extend, slots, write and trim where some tables are too short and the stack runs dry: the rows of the
    requests that were refused stay, their lengths too, and the next extension serves them from what came back."""
    gen = torch.Generator().manual_seed(requests)
    block = 4
    lengths = torch.randint(0, block * columns + 1, (requests,), generator=gen).tolist()
    while sum(ref._used(x, block, columns, False) for x in lengths) > blocks:
        lengths[lengths.index(max(lengths))] //= 2
    counts = torch.randint(0, 12, (requests,), generator=gen).tolist()
    cu, parents = trees(counts, requests)
    par = parents if tree else None
    order = torch.randperm(blocks, generator=gen).tolist()
    tables, free = [[-1] * columns for _ in lengths], order + [-1] * 3
    count = ref.extend([0] * requests, lengths, tables, free, blocks, block, sum(lengths))[2]
    last = [int(torch.randint(-1, n, (), generator=gen)) if n else -1 for n in counts]
    total, longer = cu[-1] + 5, [x + n for x, n in zip(lengths, counts)]
    keys = torch.zeros(blocks, 1, block, 8, device=gpu)
    held = torch.zeros(blocks, block, dtype=torch.bool)
    for r, x in enumerate(lengths):
        for p in range(x):
            held[tables[r][p // block], p % block] = True
    t_dev, f_dev, c_dev, l_dev = i32(tables, gpu), i32(free, gpu), i32([count], gpu), torch.tensor(lengths, device=gpu)
    par_dev = None if par is None else i32(par + [0] * 5, gpu)
    slots, served = ik.extend_block_tables(l_dev, i32(cu, gpu), t_dev, f_dev, c_dev, block, total)
    start = count
    want, serve, count = ref.extend(lengths, counts, tables, free, count, block, total)
    assert served.tolist() == serve and not all(serve) and slots.tolist() == want
    # without `last` the deepest node decides; tables that are no rings refuse by themselves past their columns
    for kw in (dict(served=served), dict(served=served, wrap=False), dict(wrap=False)):
        got, kept = ik.slot_map(i32(cu, gpu), l_dev, t_dev, block, total, parents=par_dev, **kw)
        exact = ref.slot_map(cu, lengths, tables, block, total, par, served=serve if "served" in kw else None,
                             wrap=kw.get("wrap", True))
        assert kept.tolist() == exact[1] and got.tolist() == [max(x, -1) for x in exact[0]]
    at, kept = ik.slot_map(i32(cu, gpu), l_dev, t_dev, block, total, parents=par_dev, last=i32(last, gpu), served=served)
    exact = ref.slot_map(cu, lengths, tables, block, total, par, last, serve)
    assert at.tolist() == exact[0] and kept.tolist() == exact[1]
    assert all(k == x for k, x, ok in zip(exact[1], lengths, serve) if not ok)
    layers.cache_write(torch.ones(total, 1, 8, device=gpu), torch.ones(total, 1, 8, device=gpu), at, keys, keys.clone())
    written = keys[:, 0, :, 0].cpu() > 0
    assert not (written & held).any() and int(written.sum()) == sum(exact[1]) - sum(lengths)
    ik.trim_block_tables(torch.tensor(longer, device=gpu), kept, t_dev, f_dev, c_dev, block)
    count = ref.trim(longer, exact[1], tables, free, count, block)
    assert t_dev.tolist() == tables and c_dev.item() == count <= start and f_dev[:count].tolist() == free[:count]
    for r, k in enumerate(exact[1]):     # each request holds the blocks of its length, no more and no fewer
        used = ref._used(k, block, columns, False)
        assert min(tables[r][:used], default=0) >= 0 and tables[r][used:] == [-1] * (columns - used)
    again, served = ik.extend_block_tables(kept, i32([0] + [1] * requests, gpu).cumsum(0), t_dev, f_dev, c_dev, block, requests)
    want, serve, _ = ref.extend(exact[1], [1] * requests, tables, free, count, block, requests)
    assert again.tolist() == want and served.tolist() == serve


def test_served_is_checked(gpu):
    args = (i32([0, 2], gpu), torch.tensor([1], device=gpu), i32([[0]], gpu), 4, 2)
    for bad in (torch.ones(2, dtype=torch.bool, device=gpu), torch.ones(1, dtype=torch.int32, device=gpu)):
        with pytest.raises(ValueError, match="served"):
            ik.slot_map(*args, served=bad)
    slots, kept = ik.slot_map(*args, served=torch.tensor([False]))       # from the host
    assert slots.tolist() == [-1, -1] and kept.tolist() == [1]
    assert ik.slot_map(*args, served=torch.tensor([True], device=gpu))[0].tolist() == [1, 2]


@pytest.mark.parametrize("dtype,kd,vd,most", [(torch.bfloat16, 128, 128, None), (torch.bfloat16, 128, 64, 16),
                                              (torch.bfloat16, 128, 128, 32), (torch.float32, 128, 128, None),
                                              (torch.float16, 64, 64, None)])
@pytest.mark.parametrize("chain", [True, False])
def test_delta_rule_that_forgets(gpu, dtype, kd, vd, most, chain):
    """Log decays of -inf, -3e4 and -200 among ordinary ones, one on a path and many: the state is gone there,
    as it is token by token, and the decays behind them keep their bits."""
    counts = [min(x, most or 64) for x in (64, 33, 5, 16, 1)]
    cu, parents = trees(counts, 91, back=2)
    par = None if chain else parents
    n, gen = cu[-1], torch.Generator().manual_seed(92)
    q, k = rnd(1, n, 2, kd, seed=93, dtype=dtype), rnd(1, n, 2, kd, seed=94, dtype=dtype)
    v, s0 = rnd(1, n, 4, vd, seed=95, dtype=dtype), rnd(5, 4, kd, vd, seed=96, dtype=torch.float32, std=0.3)
    beta = torch.rand(1, n, 4, generator=gen)
    g = -torch.rand(1, n, 4, generator=gen)
    kinds = torch.tensor([-float("inf"), -3e4, -200.0, -104.5, -103.0, -float("inf")])
    for head in range(4):                      # none, one in ten, half of the nodes, all
        at = torch.rand(n, generator=gen) < (0.0, 0.1, 0.5, 2.0)[head]
        g[0, at, head] = kinds[torch.randint(0, 6, (int(at.sum()),), generator=gen)]
    g[0, 0, 1] = -3e4                          # above a whole request
    got = gdn.tree_gated_delta_rule(*(x.to(gpu) for x in (q, k, v, g, beta)), None if par is None else i32(par, gpu),
                                    i32(cu, gpu), s0.to(gpu), max_nodes=most)
    want, size = ref.delta_rule(q[0], k[0], v[0], g[0], beta[0], par, cu, s0)
    within(got[0], want, half_step(dtype) * want.abs() + 2.0 ** -12 * size)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_the_accepted_paths_advance_states_and_windows(gpu, dtype):
    """The second half of a step: the conv window and the recurrent state that decoding the accepted path would
    leave, from the prefill's operators over the accepted rows; then a second draft from that state.

    The states agree with float64 as the prefill's do (1e-3 of their norm), and a float16 one is rounded once
    (2^-11).  The second draft reads such a state: its error reaches the outputs in that share of the terms."""
    s, cu, parents, lengths, block = _step(gpu, 91)
    s["state"] = s["state"].to(dtype)
    start, n = s["state"].clone(), cu[-1]
    x = layers.conv_tree(s["proj"], s["window"], s["conv_w"], s["parents"], s["cu"], 3 * 512, planes=3)
    slots, served = ik.extend_block_tables(s["lengths"], s["cu"], s["tables"], s["free"], s["count"], block, n)
    slots, kept = ik.slot_map(s["cu"], s["lengths"], s["tables"], block, n, parents=s["parents"], last=s["last"],
                              served=served)
    paths = [ref.paths(parents[a:b], b - a)[last] if last >= 0 else []
             for a, b, last in zip(cu, cu[1:], s["last"].tolist())]
    rows, cu_kept = (slots >= 0).nonzero()[:, 0], ik.cu_seqlens(kept - s["lengths"])
    assert rows.tolist() == [a + j for a, p in zip(cu, paths) for j in p] and min(map(len, paths)) == 0
    window = s["window"].clone()
    q, k, v = layers.conv_prefill(s["proj"][rows], window, s["conv_w"], cu_kept, 3 * 512, planes=3)
    for have, tree in zip((q, k, v), x):     # the rows that the draft saw
        within(have, tree[rows].double().cpu(), 2.0 ** -7 * tree[rows].double().cpu().abs() + 2.0 ** -14)
    _, new = gdn.chunk_gated_delta_rule(q.view(1, -1, 4, 128), k.view(1, -1, 4, 128), v.view(1, -1, 4, 128),
                                        g=s["g"][:, rows], beta=s["beta"][:, rows], initial_state=s["state"].float(),
                                        output_final_state=True, use_qk_l2norm_in_kernel=True, cu_seqlens=cu_kept)
    s["state"].copy_(new)
    share = 1e-3 + (2.0 ** -11 if dtype == torch.float16 else 0)
    gates, beta = s["g"][0].double().cpu(), s["beta"][0].double().cpu()
    q, k, v = (t.view(-1, 4, 128).double().cpu() for t in (q, k, v))
    k = k / torch.sqrt((k * k).sum(-1, keepdim=True) + 1e-6)
    exact, at = [], 0
    for r, path in enumerate(paths):
        taps = torch.cat((s["window"][r], s["proj"][[cu[r] + j for j in path]][:, :3 * 512]))[-3:]
        assert torch.equal(window[r], taps), r
        state = start[r].double().cpu()
        for j in path:
            state = state * torch.exp(gates[cu[r] + j])[:, None, None]
            delta = beta[cu[r] + j][:, None] * (v[at] - torch.einsum("hk,hkv->hv", k[at], state))
            state = state + k[at][:, :, None] * delta[:, None]
            at += 1
        exact.append(state)
        assert (s["state"][r].double().cpu() - state).norm() <= share * state.norm(), r
    assert at == len(rows)
    draft = [rnd(1, 40, 4, 128, seed=i).to(gpu) for i in (1, 2, 3)]
    gb = [-torch.rand(1, 40, 4, device=gpu), torch.rand(1, 40, 4, device=gpu)]
    off, par = [0, 8, 16, 24, 32, 40], trees([8] * 5, 7)[1]
    got = gdn.tree_gated_delta_rule(*draft, *gb, i32(par, gpu), i32(off, gpu), s["state"])
    want, size = ref.delta_rule(*(t[0].cpu() for t in (*draft, *gb)), par, off, torch.stack(exact))
    # decay and I - beta k k^T do not lengthen an error of the state, and q (norm 1, times scale) reads it
    reach = torch.stack([x.norm(dim=(1, 2)) for x in exact]).repeat_interleave(8, 0)[..., None] * 128 ** -0.5
    # (the bound on the state holds for all heads together: a head may have all of it)
    reach = reach.norm(dim=1, keepdim=True)
    within(got[0], want, share * reach + half_step(torch.bfloat16) * want.abs() + 2.0 ** -12 * size)


@pytest.mark.parametrize("pending", [0, 40, 59, 63])
def test_anchor_reads_of_a_draft_end_at_the_commit(gpu, pending):
    """A drafted path's reads of the memory as it is before the step are decode's reads down to the token that
    fills the chunk; the tokens behind it read another memory."""
    chunk, n = 64, 12
    memory = workloads.anchor_state(2, 2, 16, chunk, 128, seed=pending + 1, fill_pending=pending)
    state = im.IndependentMemoryState(*(getattr(memory, f.name).to(gpu) for f in fields(memory)))
    q = rnd(n, 1, 8, 128, seed=pending + 2).to(gpu)
    k, v = (rnd(n, 1, 2, 128, seed=pending + s).to(gpu) for s in (3, 4))
    draft = im.committed_gqa(q, state, i32([1] * n, gpu)).double().cpu()
    for t in range(n):
        read = im.committed_gqa(q[t:t + 1], state, i32([1], gpu)).double().cpu()[0]
        off = (draft[t] - read).norm() / read.norm()
        if t <= chunk - 1 - pending:       # two roundings to bf16, and sums in another order
            assert off <= 2 * 2.0 ** -8, t
        else:
            assert off > 0.1, t
        im.commit_decode(k[t:t + 1], v[t:t + 1], torch.full((1, 1, 2), 9.0, device=gpu), torch.tensor([True], device=gpu),
                         chunk, state, i32([1], gpu))


def test_offsets_past_the_rows_are_those_clamped(gpu):
    """Offsets below 0 and past the rows give the results of the clamped ones in every operator; offsets that
    fall give slots of the requests' own blocks or none, and take no block that is not on the stack."""
    n, block = 9, 16
    lens = torch.tensor([20, 30], device=gpu)
    x, w, proj = rnd(1, n, 2, 128, seed=5).to(gpu), rnd(2, 3, 48, seed=6).to(gpu), rnd(n, 48, seed=7).to(gpu)
    taps, g = rnd(48, 4, seed=8).to(gpu), torch.rand(1, n, 2, generator=torch.Generator().manual_seed(9)).to(gpu)
    state = rnd(2, 2, 128, 128, seed=10, dtype=torch.float32).to(gpu)
    par, last = i32([-1, 0, 0, 1, 2, -1, 0, 1, 1], gpu), i32([3, 2], gpu)

    def run(cu):
        cu, tables = i32(cu, gpu), i32([[0, 1, -1], [2, 3, -1]], gpu)
        free, count = i32([7, 5, 4, -1], gpu), i32([3], gpu)
        out = []
        for y in (x, x.float()):
            for most in (None, 8):
                out.append(gdn.tree_gated_delta_rule(y, y, y, -g, g, par, cu, state, max_nodes=most))
        for c, p in ((48, 3), (45, 1)):
            out.append(layers.conv_tree(proj, w[..., :c].contiguous(), taps[:c], par, cu, c, planes=p))
        for parents in (par, None):
            for at in (None, last):
                out += ik.slot_map(cu, lens, tables, block, n, parents=parents, last=at)
        out += ik.extend_block_tables(lens, cu, tables, free, count, block, n)
        return out + [tables, free, count]
    want = run([0, 5, 9])
    for got, exact in zip(run([-3, 5, 4000]), want):
        assert torch.equal(got, exact)
    out = run([0, 7, 3])
    tables, free, count = (t.tolist() for t in out[-3:])
    assert 0 <= count[0] <= 3 and free == [7, 5, 4, -1]
    taken = {7, 5, 4} - set(free[:count[0]])
    held = [{0, 1} | taken, {2, 3} | taken]
    for row, own in zip(tables, held):
        assert set(row) - {-1} <= own
    for slots in (*out[6:14:2], out[14]):
        assert slots.shape == (n,)
        assert all(s == -1 or s // block in {0, 1, 2, 3} | taken for s in slots.tolist())
    assert all(s == -1 or s // block in held[0] for s in out[14].tolist()[:7]) and out[14].tolist()[7:] == [-1, -1]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_many_rows_behind_the_last_request(gpu, dtype):
    """A step that is captured for its largest batch: most packed rows belong to no request.  They are zeros,
    those of the requests what they are without them, whatever was in the memory."""
    n, pad = 11, 9001
    cu = i32([0, 4, 4, n], gpu)
    q, k, v = (torch.nn.functional.pad(rnd(n, h, 128, seed=h + s), (0, 0, 0, 0, 0, pad), value=NAN).to(gpu)
               for s, h in ((1, 8), (2, 2), (3, 2)))
    cache = rnd(6, 2, 16, 128, seed=4).to(gpu)
    args = (torch.tensor([20, 3, 32], device=gpu), cache, cache, i32([[0, 1], [2, 3], [4, 5]], gpu))
    state, gates = rnd(3, 8, 128, 128, seed=5, dtype=torch.float32).to(gpu), torch.rand(1, n + pad, 8, device=gpu)
    proj, window, taps = q.reshape(n + pad, 1024), rnd(3, 3, 1024, seed=6).to(gpu), rnd(1024, 4, seed=7).to(gpu)

    def run(rows, cu):
        x = q[None, :rows].to(dtype)
        stale = [torch.full((rows, 1024), NAN, device=gpu, dtype=t) for t in (dtype, torch.bfloat16, torch.bfloat16)]
        del stale
        out = []
        for most in (None, 8):
            out.append(layers.tree_attention(q[:rows], k[:rows], v[:rows], None, cu, *args, max_nodes=most))
            out.append(gdn.tree_gated_delta_rule(x, x, x, -gates[:, :rows], gates[:, :rows], None, cu, state, max_nodes=most)[0])
        out.append(layers.conv_tree(proj[:rows], window, taps, None, cu, 1024))
        return out
    for got, want in zip(run(n + pad, cu), run(n, cu)):
        assert torch.equal(got[:n], want) and not got[n:].any()
    none = (torch.zeros(0, dtype=torch.int64, device=gpu), cache, cache, torch.zeros(0, 2, dtype=torch.int32, device=gpu))
    assert not layers.tree_attention(q, k, v, None, i32([0], gpu), *none).any()
    # outputs off 16-byte alignment, from the C call
    store, x = torch.full((1 + (n + pad) * 1024 * 4 // dtype.itemsize,), NAN, device=gpu, dtype=dtype), q.to(dtype)
    off = 2 if dtype == torch.bfloat16 else 1
    N.call_on(gpu, "yh_tree_gated_delta_rule", *[x.data_ptr()] * 3, gates.data_ptr(), gates.data_ptr(), None, cu.data_ptr(),
              state.data_ptr(), N.F32, None, store.data_ptr() + 4, 3, n + pad, 8, 8, 128, 128, 3, 64, 1.0, 1,
              N.code(x), N.F32, N.F32)
    rows = store[off:off + (n + pad) * 1024].view(n + pad, 1024)
    assert rows[:n].isfinite().all() and not rows[n:].any()
    assert store[:off].isnan().all() and store[off + (n + pad) * 1024:].isnan().all()


@pytest.mark.parametrize("n", [1, 15, 16, 17, 40])
@pytest.mark.parametrize("columns", [3, 255, 256, 257])
def test_trim_around_one_launch(gpu, n, columns):
    """Both forms of the trim where they meet: some requests whole, some in part, some not served, some longer
    than what is kept."""
    block, gen = 8, torch.Generator().manual_seed(n * columns)
    tables = torch.randperm(n * columns, generator=gen).view(n, columns).to(torch.int32)
    tables[torch.rand(n, columns, generator=gen) < 0.1] = -1
    lengths = torch.randint(0, block * columns + 1, (n,), generator=gen)
    kept = (lengths * torch.randint(0, 4, (n,), generator=gen) // 2).tolist()     # half of them as long or longer
    lengths, want = lengths.tolist(), tables.tolist()
    free = list(range(10 ** 6, 10 ** 6 + 5)) + [-1] * (n * columns)
    t_dev, f_dev, c_dev = tables.to(gpu), i32(free, gpu), i32([5], gpu)
    ik.trim_block_tables(torch.tensor(lengths, device=gpu), torch.tensor(kept, device=gpu), t_dev, f_dev, c_dev, block)
    count = ref.trim(lengths, kept, want, free, 5, block)
    assert t_dev.tolist() == want and c_dev.item() == count and f_dev.tolist() == free
