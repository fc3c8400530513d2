"""Drafted trees without a GPU: the oracle against the package's sequential
oracles, what the wrappers and the C calls refuse, and block bookkeeping laws."""
import ctypes

import pytest
import torch

from oracle import gdn as seq
from oracle import tree as ref
from yanchor_amd import _native, _tree, gdn, layers
from yanchor_amd import inference_kernels as ik


def test_paths():
    assert ref.paths([-1, 0, 0, 1, -1, 4], 6) == [[0], [0, 1], [0, 2], [0, 1, 3], [4], [4, 5]]
    assert ref.paths(None, 3) == [[0], [0, 1], [0, 1, 2]]
    assert ref.paths([0, 5, -7], 3) == [[0], [1], [2]]      # no earlier node: the context


def test_chain_delta_rule_is_the_recurrence():
    torch.manual_seed(1)
    t, h, hv, d = 5, 2, 4, 8
    q, k, v = torch.randn(1, t, h, d), torch.randn(1, t, h, d), torch.randn(1, t, hv, d)
    g, beta, s = -torch.rand(1, t, hv), torch.rand(1, t, hv), torch.randn(1, hv, d, d)
    o, _ = seq.recurrent_gated_delta_rule(q.double(), k.double(), v.double(), g.double(), beta.double(), s.double())
    mine, _ = ref.delta_rule(q[0], k[0], v[0], g[0], beta[0], None, [0, t], s)
    assert torch.allclose(mine, o[0], rtol=1e-10, atol=1e-12)   # both in float64


@pytest.mark.parametrize("wrap", [False, True])
def test_trim_takes_an_extension_back(wrap):
    lengths, added = [0, 5, 16, 3], [7, 0, 20, 1]
    tables = [[-1] * 6 for _ in lengths]
    free = list(range(40, 60))
    _, served, count = ref.extend([0] * 4, lengths, tables, free, len(free), 4, 24, wrap)
    assert all(served)
    before = ([list(t) for t in tables], list(free), count)
    slots, served, count = ref.extend(lengths, added, tables, free, count, 4, 30, wrap)
    # request 2 would need 9 columns: it is served only where they are a ring
    assert served == [True, True, wrap, True] and slots[28:] == [-1, -1] and (wrap or slots[7:27] == [-1] * 20)
    count = ref.trim([a + b for a, b in zip(lengths, added)], lengths, tables, free, count, 4, wrap)
    assert (tables, count) == (before[0], before[2]) and free[:count] == before[1][:count]


def test_an_empty_stack_serves_no_later_request():
    tables = [[-1] * 4 for _ in range(4)]
    slots, served, count = ref.extend([0, 0, 0, 2], [4, 12, 4, 1], tables, [9, 8, 7], 3, 4, 21)
    assert served == [True, False, False, True] and count == 2     # the last needs no block


@pytest.mark.parametrize("length,added", [(0, 30), (5, 8), (7, 9), (20, 17), (3, 0)])
def test_a_ring_keeps_the_last_of_a_row(length, added):
    block, columns = 4, 2
    tables, free = [[-1] * columns], [7, 5]
    ref.extend([0], [length], tables, free, 2, block, length, True)
    used = sum(x >= 0 for x in tables[0])
    slots, served, _ = ref.extend([length], [added], tables, free, 2 - used, block, added, True)
    rows = [x for x in slots if x >= 0]
    assert served == [True] and len(set(rows)) == len(rows) == min(added, block * columns)
    assert slots[:added - len(rows)] == [-1] * (added - len(rows))
    again, _ = ref.slot_map([0, added], [length], tables, block, added)
    assert again == slots


# --- refusals: nothing reaches a device ---------------------------------------

def _attn(**kw):
    a = dict(q=torch.zeros(4, 8, 128, dtype=torch.bfloat16), k=torch.zeros(4, 2, 128, dtype=torch.bfloat16),
             v=torch.zeros(4, 2, 128, dtype=torch.bfloat16), parents=None, cu_seqlens=torch.tensor([0, 4]),
             lengths=torch.tensor([3]), keys=torch.zeros(2, 2, 16, 128, dtype=torch.bfloat16),
             values=torch.zeros(2, 2, 16, 128, dtype=torch.bfloat16),
             block_tables=torch.zeros(1, 2, dtype=torch.int32))
    a.update(kw)
    return layers.tree_attention(**a)


@pytest.mark.parametrize("kw,match", [
    (dict(q=torch.zeros(4, 8, 128)), "one dtype"),
    (dict(q=torch.zeros(4, 7, 128, dtype=torch.bfloat16)), "dividing"),
    (dict(q=torch.zeros(4, 8, 96, dtype=torch.bfloat16), k=torch.zeros(4, 2, 96, dtype=torch.bfloat16),
          v=torch.zeros(4, 2, 96, dtype=torch.bfloat16)), "64 or 128"),
    (dict(keys=torch.zeros(2, 3, 16, 128, dtype=torch.bfloat16)), "contiguous"),
    (dict(values=torch.zeros(2, 2, 16, 128, dtype=torch.float16)), "contiguous"),
    (dict(), "ROCm device"),
])
def test_attention_refuses(kw, match):
    with pytest.raises(ValueError, match=match):
        _attn(**kw)


def test_host_offsets_are_checked():
    dev = torch.device("cpu")
    assert _tree.offsets(torch.tensor([0, 2, 2, 5]), 6, dev).tolist() == [0, 2, 2, 5]
    for bad in ([1, 3], [0, 4, 2], [0, 9]):
        with pytest.raises(ValueError, match="offsets"):
            _tree.offsets(torch.tensor(bad), 6, dev)
    with pytest.raises(ValueError, match="at most 64"):
        _tree.nodes(None, torch.tensor([0, 65]), None, 65, dev)
    with pytest.raises(ValueError, match="1 to 64"):
        _tree.nodes(None, torch.tensor([0, 5]), 65, 5, dev)
    with pytest.raises(ValueError, match="5 entries"):
        _tree.nodes(torch.zeros(4, dtype=torch.int32), torch.tensor([0, 5]), 8, 5, dev)
    with pytest.raises(ValueError, match="integer"):
        _tree.nodes(torch.zeros(5), torch.tensor([0, 5]), 8, 5, dev)


def test_the_other_wrappers_refuse_host_tensors():
    b = torch.bfloat16
    i32 = dict(dtype=torch.int32)
    tables, free, count = torch.zeros(1, 2, **i32), torch.zeros(4, **i32), torch.zeros(1, **i32)
    one, cu = torch.tensor([1]), torch.tensor([0, 1])
    with pytest.raises(ValueError, match="ROCm device"):
        ik.extend_block_tables(one, cu, tables, free, count, 16, 1)
    with pytest.raises(ValueError, match="ROCm device"):
        ik.trim_block_tables(one, one, tables, free, count, 16)
    with pytest.raises(ValueError, match="ROCm device"):
        ik.slot_map(cu, one, tables, 16, 1)
    k, cache = torch.zeros(1, 2, 64, dtype=b), torch.zeros(2, 2, 16, 64, dtype=b)
    with pytest.raises(ValueError, match="ROCm device"):
        layers.cache_write(k, k, one, cache, cache)
    with pytest.raises(ValueError, match="16 bytes"):
        layers.cache_write(k[..., :4], k[..., :4], one, cache, cache)
    with pytest.raises(ValueError, match="ROCm device"):
        layers.conv_tree(torch.zeros(1, 24, dtype=b), torch.zeros(1, 3, 24, dtype=b), torch.zeros(24, 4, dtype=b), None,
                         cu, 24)
    x, gate = torch.zeros(1, 1, 2, 128, dtype=b), torch.zeros(1, 1, 2)
    state = torch.zeros(1, 2, 128, 128)
    with pytest.raises(ValueError, match="ROCm device"):
        gdn.tree_gated_delta_rule(x, x, x, gate, gate, None, cu, state)
    with pytest.raises(ValueError, match="64 or 128"):
        gdn.tree_gated_delta_rule(x[..., :96], x[..., :96], x, gate, gate, None, cu, state)
    with pytest.raises(ValueError, match="do not match"):
        gdn.tree_gated_delta_rule(x, x, x, gate[..., :1], gate, None, cu, state)


@pytest.fixture(scope="module")
def lib():
    return _native.lib()


def test_c_calls_refuse_before_device_work(lib):
    p = ctypes.c_void_p(256)
    odd = ctypes.c_void_p(264)

    def refused(rc, text):
        assert rc == -1 and text in lib.yh_last_error(), lib.yh_last_error()

    def attn(q=p, d=128, block=16, max_nodes=64, qs=1024, cu=p, gate=None, ghs=0, dtype=1, blocks=2, total=4, ws=1 << 30):
        return lib.yh_tree_attention(q, qs, p, 256, p, 256, None, cu, p, p, p, p, gate, 1024, ghs, p, 1, total, blocks, 2,
                                     8, 2, d, block, 0, max_nodes, -1, 1.0, dtype, p, ws, None)
    refused(attn(d=96), b"64 or 128")
    refused(attn(block=0), b"bad sizes")
    refused(attn(max_nodes=65), b"max_nodes")
    refused(attn(cu=None), b"null")
    refused(attn(q=odd), b"aligned")
    refused(attn(qs=512), b"whole heads")
    refused(attn(gate=p, ghs=64), b"gate strides")
    refused(attn(blocks=1 << 28), b"too large")
    refused(attn(ws=lib.yh_tree_attention_workspace_bytes(1, 8, 2, 128, 16, 2, 0, 64, -1) - 1), b"workspace")
    assert attn(dtype=0) == -3
    assert attn(total=0) == 0

    refused(lib.yh_extend_block_tables(p, p, p, p, p, p, p, p, 1, 0, 4, 4, 16, 0, None), b"bad sizes")
    refused(lib.yh_extend_block_tables(None, p, p, p, p, p, p, p, 1, 1, 4, 4, 16, 0, None), b"null")
    refused(lib.yh_extend_block_tables(p, p, p, p, p, p, p, p, 0, 1, 4, 4, 16, 0, None), b"without requests")
    assert lib.yh_extend_block_tables(None, None, None, None, None, None, None, None, 0, 1, 0, 0, 16, 0, None) == 0
    refused(lib.yh_trim_block_tables(p, p, p, p, None, p, 1, 1, 4, 16, 0, None), b"null")
    refused(lib.yh_trim_block_tables(p, p, p, p, p, p, 1, 1, 4, 0, 0, None), b"bad sizes")
    refused(lib.yh_slot_map(p, p, None, None, None, p, p, 1, 1, 4, 16, None), b"null")
    refused(lib.yh_cache_write(p, 128, p, 128, p, p, p, None, None, 4, 2, 1, 100, 16, 1, None), b"16 bytes")
    refused(lib.yh_cache_write(odd, 128, p, 128, p, p, p, None, None, 4, 2, 1, 128, 16, 1, None), b"aligned")
    refused(lib.yh_cache_write(p, 128, p, 128, p, p, p, p, None, 4, 2, 1, 128, 16, 1, None), b"come together")
    refused(lib.yh_cache_write(p, 128, p, 128, p, p, p, None, None, 4, 2, 1, 128, 16, 3, None), b"dtype")

    def delta(k=128, hv=4, rows=1, idx=None, st=0, max_nodes=64):
        return lib.yh_tree_gated_delta_rule(p, p, p, p, p, None, p, p, st, idx, p, 2, 4, 2, hv, k, 128, rows, max_nodes,
                                            1.0, 1, 1, 0, 0, None)
    refused(delta(k=96), b"64 or 128")
    refused(delta(hv=3), b"multiple")
    refused(delta(), b"fewer state rows")
    refused(delta(rows=2, st=1), b"f32 or f16")
    refused(delta(rows=2, max_nodes=0), b"max_nodes")
    refused(lib.yh_conv_tree(p, 24, p, p, None, p, 1, 4, 24, 5, p, 1, None), b"divide")
    refused(lib.yh_conv_tree(p, 23, p, p, None, p, 1, 4, 24, 1, p, 1, None), b"bad sizes")
    refused(lib.yh_conv_tree(p, 24, p, p, None, p, 1, 4, 24, 1, p, 0, None), b"bfloat16")


@pytest.mark.parametrize("table,free", [([5, 6], [9]), ([5, 6, -1], [])])
def test_a_refused_request_gets_no_slots(table, free):
    """Too few columns, or a dry stack: nothing is written, the length stays."""
    tables = [list(table), [7] + [-1] * (len(table) - 1)]
    slots, served, count = ref.extend([7, 1], [4, 2], tables, list(free), len(free), 4, 6)
    assert served == [False, True] and slots == [-1] * 4 + [29, 30]
    for par in (None, [-1, 0, 1, 2, -1, 0]):
        for last, kept in ((None, 3), ([3, 0], 2)):
            got = ref.slot_map([0, 4, 6], [7, 1], tables, 4, 6, par, last, served)
            assert got == ([-1] * 4 + [29, 30 if last is None else -1], [7, kept])
    # without `served` a table that is no ring at least does not start over
    if len(table) == 2:
        assert ref.slot_map([0, 4, 6], [7, 1], tables, 4, 6, wrap=False) == ([-1] * 4 + [29, 30], [7, 3])
        assert ref.slot_map([0, 4, 6], [7, 1], tables, 4, 6)[0][:4] == [27, 20, 21, 22]      # a ring does


def test_served_slots_refuse_before_device_work(lib):
    p = ctypes.c_void_p(256)
    assert lib.yh_slot_map_served(p, p, None, None, None, p, p, p, 1, 1, 4, 16, 0, None) == -1
    assert b"null" in lib.yh_last_error()
    assert lib.yh_slot_map_served(p, p, p, None, None, p, p, p, 1, 0, 4, 16, 0, None) == -1
    assert b"bad sizes" in lib.yh_last_error()
    assert lib.yh_slot_map_served(None, None, None, None, None, None, None, None, 0, 1, 0, 16, 0, None) == 0


def test_the_recurrence_refuses_packed_sequences():
    """It has no offsets: the requests' tokens would run one after another into the first state row."""
    x, gate = torch.zeros(1, 5, 2, 128, dtype=torch.bfloat16), torch.zeros(1, 5, 2)
    for f in (gdn.recurrent_gated_delta_rule, gdn.fused_recurrent_gated_delta_rule):
        with pytest.raises(ValueError, match="chunk_gated_delta_rule"):
            f(x, x, x, g=gate, beta=gate, initial_state=torch.zeros(2, 2, 128, 128), cu_seqlens=torch.tensor([0, 3, 5]))
        for one in (None, torch.tensor([0, 5])):       # as ever: a single sequence
            with pytest.raises(ValueError, match="ROCm device"):
                f(x, x, x, g=gate, beta=gate, initial_state=torch.zeros(1, 2, 128, 128), cu_seqlens=one)
