"""Decoding over a quantised block cache on the GPU, against float64.

Tolerances, from the roundings that each kernel makes (e = half a step of a type,
torch.finfo(t).eps / 2):
* quantised rows are exact: the scales are powers of two and the codes are
  rounded from exact quotients.
* attention: the output is rounded once (e |o|).  Weights that enter the value
  product rounded once to its type are off by e sum p |v|, as a pair by 2^-16: the
  kernel takes pairs, most bounds here allow the one rounding (bf16 for bf16
  queries, fp16 for a 16-bit fp16 cache), and the tests of equal weights do not.  Scores, exponentials and sums are float32: the error of a
  score (256 terms, 2^-24 each, of scores up to some tens, a capped one 2^-22 of
  its cap, a bias 2^-24 of its size) leaves 2^-12 sum p |v|.
* norms and rotations: the output once (e |o|); the norm (2^-22), the angle
  (2^-25 of a turn) and the products leave 2^-18 of the pair's magnitudes.
* an output below the type's normal numbers is rounded to a multiple of the
  smallest subnormal, smallest_normal x eps: half of that (fp16 2^-25, bf16
  2^-134) may be lost whatever its size.  (Four-bit values are often 0, so that
  an output can be all of it keys of tiny weights.)
"""
import math

import pytest
import torch

from oracle import qcache as ref
from yanchor_amd import inference_kernels as ik
from yanchor_amd import _native as N
from yanchor_amd import layers

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")
B, H16 = torch.bfloat16, torch.float16


def half_step(t):
    return torch.finfo(t).eps / 2


def within(x, want, bound, what=""):
    """|x - want| <= bound, and half of the smallest subnormal, everywhere; the worst ratio is told."""
    bound = bound + torch.finfo(x.dtype).smallest_normal * half_step(x.dtype)
    x = x.detach().double().cpu()
    assert x.shape == want.shape
    bad = ~((x - want).abs() <= bound + 1e-30)
    ratio = ((x - want).abs() / (bound + 1e-30)).max().item() if x.numel() else 0
    assert not bad.any(), f"{what}: {int(bad.sum())} of {x.numel()} off, {ratio:.2f} times the bound, first at {bad.nonzero()[0].tolist()}"


def rnd(*shape, seed, dtype=B, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def cache_of(x, y, bits):
    """A quantised cache on the CPU that holds keys x and values y [blocks, G, block, D], by the oracle."""
    blocks, g, block, d = x.shape
    c = layers.quantized_cache(blocks, g, block, d, bits=bits, device="cpu")
    table = ref.code_values(bits)
    n = len(table) // 2
    mags = table[:n][~table[:n].isnan()]
    for which, t in enumerate((x, y)):
        val, s = ref.quantise(t, bits)
        unit = torch.where(s == 255, 1.0, 2.0 ** (s.double() - 127)).repeat_interleave(32, -1)
        v = (val / unit).nan_to_num(0.0)
        code = (torch.searchsorted(mags, v.abs()) + n * (v < 0)).to(torch.uint8)
        if bits == 4:
            code = code[..., ::2] + 16 * code[..., 1::2]
        c[which].view(torch.uint8).copy_(code)
        c[2 + which].copy_(s.transpose(2, 3))
    return c


# --- write and read ---------------------------------------------------------------

def odd_rows(n, g, d, dtype, seed):
    """Rows with runs of zeros, of tiny and huge values, of codes' borders, of NaN and infinities."""
    x = rnd(n, g, d, seed=seed, dtype=torch.float32)
    big = 4.0 if dtype == H16 else 100.0
    x *= torch.exp2(torch.randint(-int(big), int(big), (n, g, 1), generator=torch.Generator().manual_seed(seed)).float())
    if n > 12:
        x[0, 0] = 0
        x[1, 0, :32] = torch.arange(32) / 32 * 6          # ties of both types
        x[2, 0, :32] = torch.arange(32) / 16 * 448 / 2
        x[3, 0, 5], x[4, 0, 7], x[5, 0, 0] = INF, NAN, -INF
        x[6, 0, 1] = torch.finfo(dtype).max
        x[7, 0, 2] = -torch.finfo(dtype).max / 2
        x[8, 0, :32] = torch.finfo(dtype).smallest_normal / 8
        x[9, 0, :32] = 2.0 ** -24 if dtype == H16 else 2.0 ** -120
        x[10, 0, :32] = -0.0
        x[11, 0, :32] = 1.75 * 2.0 ** -9
        x[12, 0, :32] = torch.linspace(-6, 6, 32)
    return x.to(dtype)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [B, H16])
@pytest.mark.parametrize("n,g,d,block", [(1, 1, 32, 1), (3, 2, 64, 16), (130, 5, 96, 7), (257, 8, 128, 64),
                                         (40, 3, 256, 1024)])
def test_write_and_read_back(gpu, bits, dtype, n, g, d, block):
    k, v = odd_rows(n, g, d, dtype, n), odd_rows(n, g, d, dtype, n + 1)
    blocks = -(-n // block) + 2
    gen = torch.Generator().manual_seed(n)
    slots = torch.randperm(blocks * block, generator=gen)[:n]
    slots[torch.rand(n, generator=gen) < 0.2] = -1
    if n > 2:
        slots[1], slots[2] = blocks * block, -7
    cache = [x.to(gpu) for x in layers.quantized_cache(blocks, g, block, d, bits=bits, device="cpu")]
    for x in cache:
        x.view(torch.uint8).fill_(0x5a)
    before = [x.view(torch.uint8).cpu() for x in cache]
    wide = torch.zeros(n, 2 * g * d + 8, dtype=dtype, device=gpu)
    wide[:, 8:8 + g * d], wide[:, 8 + g * d:] = k.to(gpu).view(n, -1), v.to(gpu).view(n, -1)
    layers.cache_write_quantized(wide[:, 8:8 + g * d].view(n, g, d), wide[:, 8 + g * d:].view(n, g, d), slots.to(gpu),
                                 *cache)
    on = [x.view(torch.uint8).cpu() for x in cache]
    live = ((slots >= 0) & (slots < blocks * block)).nonzero().flatten().tolist()
    used = torch.zeros(blocks, block, dtype=torch.bool)
    for which, x in enumerate((k, v)):
        val, s = ref.quantise(x, bits)
        got = ref.cache_values(on[which] if bits == 4 else on[which].view(torch.float8_e4m3fn), on[2 + which])
        for i in live:
            b, row = divmod(int(slots[i]), block)
            used[b, row] = True
            assert torch.equal(on[2 + which][b, :, :, row], s[i]), i
            assert torch.equal(got[b, :, row].nan_to_num(12345.0), val[i].nan_to_num(12345.0)), i
        assert torch.equal(on[which].transpose(1, 2)[~used], before[which].transpose(1, 2)[~used])
        assert torch.equal(on[2 + which].permute(0, 3, 1, 2)[~used], before[2 + which].permute(0, 3, 1, 2)[~used])
    for out in (dtype, H16 if dtype == B else B):
        rows = layers.cache_read(slots.to(gpu), *cache, dtype=out)
        for x, row in zip((k, v), rows):
            want = ref.quantise(x, bits)[0]
            dead = torch.ones(n, dtype=torch.bool)
            dead[live] = False
            want[dead] = 0
            assert torch.equal(row.cpu().nan_to_num(12345.0, 54321.0, -54321.0),
                               want.to(out).nan_to_num(12345.0, 54321.0, -54321.0))


@pytest.mark.parametrize("bits", [8, 4])
def test_read_every_code_and_scale(gpu, bits):
    """All codes under the scales that are written, from 2^-111 on, and NaN."""
    table = ref.code_values(bits)
    codes = torch.arange(256).to(torch.uint8)
    row = codes.view(-1, 32 if bits == 8 else 16)          # runs of 32 values
    scales = torch.tensor([16, 17, 100, 126, 127, 128, 140, 200, 240, 247, 255], dtype=torch.uint8)
    n, d = len(scales), 32 * len(row)
    keys = codes.view(1, 1, 1, -1).expand(n, 1, 1, -1).contiguous()
    s = scales.view(n, 1, 1, 1).expand(n, 1, d // 32, 1).contiguous()
    keys = keys.view(torch.float8_e4m3fn) if bits == 8 else keys
    got = layers.cache_read(torch.arange(n, device=gpu), keys.to(gpu), keys.to(gpu), s.to(gpu), s.to(gpu))
    for x in got:
        want = ref.cache_values(keys, s)[:, :, 0].to(B)
        assert torch.equal(x.cpu().nan_to_num(7777.0), want.nan_to_num(7777.0))
    assert table.numel() == 1 << bits


@pytest.mark.parametrize("dtype,d", [(B, 128), (H16, 8), (B, 72)])
def test_read_16_bit_rows(gpu, dtype, d):
    keys, values = (rnd(5, 3, 7, d, seed=s, dtype=dtype) for s in (1, 2))
    slots = torch.tensor([34, 0, -1, 35, 8, 8, 1 << 40, 20])
    for dt in (None, dtype):
        k, v = layers.cache_read(slots.to(gpu), keys.to(gpu), values.to(gpu), dtype=dt)
        for x, c in ((k, keys), (v, values)):
            for i, s in enumerate(slots.tolist()):
                want = c[s // 7, :, s % 7] if 0 <= s < 35 else torch.zeros(3, d, dtype=dtype)
                assert torch.equal(x[i].cpu(), want)


def test_empty_calls(gpu):
    none = torch.zeros(0, dtype=torch.int64, device=gpu)
    for bits in (4, 8):
        c = layers.quantized_cache(2, 2, 16, 64, bits=bits, device=gpu)
        z = torch.zeros(0, 2, 64, dtype=B, device=gpu)
        layers.cache_write_quantized(z, z, none, *c)
        assert layers.cache_read(none, *c)[0].shape == (0, 2, 64)
        e = layers.quantized_cache(0, 2, 16, 64, bits=bits, device=gpu)
        one = torch.ones(1, 2, 64, dtype=B, device=gpu)
        layers.cache_write_quantized(one, one, none.new_zeros(1), *e)
        assert not layers.cache_read(none.new_zeros(1), *e)[1].any()
        out = layers.decode_attention(torch.zeros(0, 4, 64, dtype=B, device=gpu), c[0], c[1], i32([[0]], gpu)[:0], none,
                                      key_scales=c[2], value_scales=c[3])
        assert out.shape == (0, 4, 64)
        out = layers.decode_attention(one, e[0], e[1], i32([[0, 3]], gpu), none.new_full((1,), 20), key_scales=e[2],
                                      value_scales=e[3])
        assert not out.any()       # no block is there: nothing is seen
    q = torch.zeros(0, 2, 64, dtype=B, device=gpu)
    out = layers.qk_norm_rope(q, q, None, None, none, torch.ones(8, device=gpu), 1e-6)
    assert out[0].shape == out[1].shape == (0, 2, 64)


# --- attention --------------------------------------------------------------------

def attention_case(dev, lengths, *, bits=8, dtype=B, h=8, g=2, d=128, block=16, columns=None, seed=0, bad=None, std=1.5,
                   gate=None, starts=None, slopes=None, strided=False, fill=0xff, **kw):
    r = len(lengths)
    columns = columns or max(1, max(-(-x // block) for x in lengths))
    blocks = r * columns + 2
    order = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed)).tolist()
    x, y = (rnd(blocks, g, block, d, seed=seed + s, dtype=dtype) for s in (1, 2))
    tables = torch.full((r, columns), -1, dtype=torch.int32)
    live = torch.zeros(blocks, block, dtype=torch.bool)
    for i, n in enumerate(lengths):
        for p in range(max(0, n - columns * block), n):
            c = p // block % columns
            tables[i, c] = order[i * columns + c]
            live[tables[i, c], p % block] = True
    if bits == 16:
        cache = [x, y, None, None]
        for t in cache[:2]:
            t.transpose(1, 2)[~live] = NAN if fill == 0xff else 0
    else:
        cache = list(cache_of(x, y, bits))
        for t in cache[:2]:      # what no position holds may be anything
            t.view(torch.uint8).transpose(1, 2)[~live] = fill
        for t in cache[2:]:
            t.permute(0, 3, 1, 2)[~live] = fill
    full = [ref.cache_values(cache[i], cache[2 + i]) for i in range(2)]
    for i, c, t in bad or []:
        tables[i, c] = t
    q = rnd(r, h, d, seed=seed + 3, dtype=dtype, std=std)
    gt = rnd(r, h, 2 * d + 1, seed=seed + 4, dtype=dtype)[:, :, d:2 * d] if gate else None
    sl = None if slopes is None else torch.tensor(slopes, dtype=torch.float32)
    to = lambda t: None if t is None else t.to(dev)  # noqa: E731
    qd = q.to(dev)
    if strided:
        wide = torch.full((r, h * d + 24), NAN, dtype=dtype, device=dev)
        wide[:, 8:8 + h * d] = qd.view(r, -1)
        qd = wide[:, 8:8 + h * d].view(r, h, d)
    got = layers.decode_attention(
        qd, to(cache[0]), to(cache[1]), to(tables), torch.tensor(lengths, device=dev), key_scales=to(cache[2]),
        value_scales=to(cache[3]), starts=None if starts is None else torch.tensor(starts, device=dev), slopes=to(sl),
        gate=None if gt is None else torch.empty_strided(gt.shape, gt.stride(), dtype=dtype, device=dev).copy_(gt), **kw)
    kw.pop("max_length", None)
    want, size = ref.attention(q, *full, tables, lengths, starts=starts, slopes=sl, gate=gt, **kw)
    p_step = 2.0 ** -16 if dtype == H16 and bits < 16 else half_step(dtype)
    within(got, want, half_step(dtype) * want.abs() + (p_step + 2.0 ** -12) * size, (bits, dtype, d))
    return got


FORMS = [(8, B), (4, B), (16, B), (8, H16), (4, H16), (16, H16)]


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("bits,dtype", FORMS)
def test_attention_lengths(gpu, bits, dtype, d):
    attention_case(gpu, [0, 1, 2, 15, 16, 17, 63, 64, 65, 255, 256, 257, 300], bits=bits, dtype=dtype, d=d, seed=1)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("bits,dtype", FORMS)
@pytest.mark.parametrize("block", [1, 24])
def test_attention_odd_blocks(gpu, bits, dtype, d, block):
    attention_case(gpu, [0, 1, 23, 24, 25, 130, 64], bits=bits, dtype=dtype, d=d, block=block, h=4, seed=2)


@pytest.mark.parametrize("h,g,block", [(1, 1, 16), (6, 2, 48), (5, 1, 8), (16, 1, 64), (17, 1, 16), (40, 2, 32),
                                       (71, 1, 16), (8, 8, 256)])
@pytest.mark.parametrize("bits", [8, 4])
def test_attention_heads_and_blocks(gpu, bits, h, g, block):
    attention_case(gpu, [70, 5, 300], bits=bits, h=h, g=g, block=block, d=64, seed=3)


@pytest.mark.parametrize("window,block,columns", [(1, 16, None), (3, 16, None), (100, 16, 8), (64, 64, 1), (40, 40, 1),
                                                  (50, 24, 3), (1000, 16, None)])
@pytest.mark.parametrize("bits", [8, 16])
def test_attention_windows_and_rings(gpu, bits, window, block, columns):
    attention_case(gpu, [0, 39, 40, 41, 300, 1000, 64], bits=bits, window=window, block=block, columns=columns, seed=4)


def test_attention_reads_the_last_positions_that_are_there(gpu):
    attention_case(gpu, [100, 48, 49, 47], block=16, columns=3, seed=5)


@pytest.mark.parametrize("bits", [8, 4, 16])
def test_attention_documents(gpu, bits):
    """Starts within, at and past the end, before the first position, beside a window."""
    attention_case(gpu, [100, 64, 64, 300, 20, 7, 90], bits=bits, starts=[50, 63, 64, 299, 500, -4, 0], seed=6)
    attention_case(gpu, [100, 64, 200, 300], bits=bits, starts=[97, 0, 150, 20], window=20, seed=7)


@pytest.mark.parametrize("bits,dtype", FORMS)
def test_attention_caps_biases_and_gates(gpu, bits, dtype):
    lengths = [33, 90, 500, 1]
    slopes = [2.0 ** -(i + 1) for i in range(8)]
    attention_case(gpu, lengths, bits=bits, dtype=dtype, softcap=15.0, gate=True, seed=8)
    attention_case(gpu, lengths, bits=bits, dtype=dtype, slopes=slopes, strided=True, seed=9)
    attention_case(gpu, lengths, bits=bits, dtype=dtype, slopes=slopes, softcap=3.0, window=77, gate=True, scale=0.5,
                   starts=[3, 0, 10, 0], strided=True, seed=10)


def test_attention_slopes_of_both_signs_and_none(gpu):
    slopes = [-0.01, 0.0, 0.5, -0.0, 1.0, 3.0, 0.001, -20.0]
    attention_case(gpu, [70, 300], slopes=slopes, seed=11)
    # biases of up to 10^5 over the length: only those near the end that has the least count
    attention_case(gpu, [5000, 4000], slopes=slopes, starts=[0, 1500], window=3900, softcap=20.0, d=64, seed=11)


@pytest.mark.parametrize("cap", [0.01, 1.0, 3e4, 1e8])
def test_attention_caps_of_any_size(gpu, cap):
    """Scores far past the cap, and a cap far past the scores, which then are what they were."""
    attention_case(gpu, [300, 40], softcap=cap, seed=21)


@pytest.mark.parametrize("bits,dtype", FORMS)
def test_attention_long_caches_in_parts(gpu, bits, dtype):
    attention_case(gpu, [5000, 70, 900, 0, 2049], bits=bits, dtype=dtype, h=4, g=2, seed=12)
    attention_case(gpu, [9000], bits=bits, dtype=dtype, h=2, g=1, d=64, block=64, softcap=20.0, gate=True, seed=13)


def test_attention_long_odd_blocks_heads_and_windows(gpu):
    attention_case(gpu, [3001, 1500], h=20, g=1, d=64, block=24, seed=14)
    attention_case(gpu, [3001, 1500, 40], bits=4, h=4, g=2, d=256, window=2000, starts=[1200, 0, 39], seed=15)


def test_attention_of_many_requests(gpu):
    """More requests than a workgroup has threads, most short, some idle, two long ones."""
    gen = torch.Generator().manual_seed(1)
    lengths = torch.randint(0, 60, (700,), generator=gen).tolist()
    lengths[3], lengths[600], lengths[699] = 2000, 1500, 0
    attention_case(gpu, lengths, h=2, g=1, d=64, block=32, seed=16)


@pytest.mark.parametrize("requests,h,g", [(130, 2, 1), (40, 8, 8), (64, 20, 1), (65, 4, 4)])
@pytest.mark.parametrize("bits", [8, 16])
def test_attention_of_many_requests_in_parts(gpu, bits, requests, h, g):
    """Some cut and some not, found by a wave (64 requests) and by a workgroup (65), parts of several turns."""
    gen = torch.Generator().manual_seed(requests)
    lengths = torch.randint(0, 900, (requests,), generator=gen).tolist()
    lengths[2], lengths[-1], lengths[requests // 2] = 3300, 2500, 0
    attention_case(gpu, lengths, bits=bits, h=h, g=g, d=64, block=48, seed=22)


@pytest.mark.parametrize("max_length", [None, 10, 250, 5000])
def test_attention_bounds_change_nothing(gpu, max_length):
    """A bound that is too low changes no result."""
    attention_case(gpu, [40, 250, 0, 1000], h=4, g=2, d=64, seed=17, max_length=max_length)


def test_attention_holes_in_a_table_are_not_seen(gpu):
    for bits, block in ((8, 16), (4, 16), (16, 16), (8, 24), (16, 1)):
        col = 200 // block
        attention_case(gpu, [200, 130, 16], bits=bits, block=block, seed=18,
                       bad=[(0, 3, -1), (0, col - 1, 1 << 30), (1, 0, 10 ** 6), (1, 1, -5), (2, 0, -1)])


def test_attention_of_an_empty_table(gpu):
    got = attention_case(gpu, [16, 40], bad=[(0, 0, -1), (1, 0, -1), (1, 1, -2), (1, 2, 999)], seed=19)
    assert not got.any()


@pytest.mark.parametrize("bits,dtype", FORMS)
def test_attention_large_scores(gpu, bits, dtype):
    """Scores of several hundred: the softmax is nearly one key."""
    attention_case(gpu, [150, 700], bits=bits, dtype=dtype, scale=1.0, seed=20, h=4)


@pytest.mark.parametrize("bits", [8, 16])
def test_attention_of_many_small_weights(gpu, bits):
    """One key of score 13 among 20000 of none: e^-13 each, in sum a twentieth of the weight, which fp16 would
    lose below 2^-24 of the largest."""
    n, d = 20000, 64
    x = torch.zeros(n // 16, 1, 16, d, dtype=H16)
    x[100, 0, 3] = 13 / 8
    y = torch.ones(n // 16, 1, 16, d, dtype=H16)
    y[100, 0, 3] = 0
    q = torch.ones(1, 1, d, dtype=H16)
    cache = list(cache_of(x, y, 8)) if bits == 8 else [x, y, None, None]
    full = [ref.cache_values(cache[i], cache[2 + i]) for i in range(2)]
    tables = torch.arange(n // 16, dtype=torch.int32)[None]
    on = [None if t is None else t.to(gpu) for t in cache]
    got = layers.decode_attention(q.to(gpu), on[0], on[1], tables.to(gpu), torch.tensor([n], device=gpu),
                                  key_scales=on[2], value_scales=on[3])
    want, size = ref.attention(q, *full, tables, [n])
    assert 0.01 < want[0, 0, 0] < 0.1
    within(got, want, (2 * half_step(H16) + 2.0 ** -12) * size)


@pytest.mark.parametrize("bits,dtype", FORMS)
@pytest.mark.parametrize("what", [NAN, INF])
def test_attention_keeps_what_is_not_finite_to_those_that_see_it(gpu, bits, dtype, what):
    lengths, d, g, h = [100, 90, 64], 128, 2, 8
    x, y = (rnd(21, g, 16, d, seed=s, dtype=dtype) for s in (1, 2))
    tables = torch.arange(21, dtype=torch.int32).view(3, 7)
    y[0, 0, 9, 3] = what          # request 0, position 9, group 0
    x[7 + 5, 1, 3, 40] = NAN      # request 1, position 83, group 1
    cache = list(cache_of(x, y, bits)) if bits < 16 else [x, y, None, None]
    on = [None if t is None else t.to(gpu) for t in cache]
    q = rnd(3, h, d, seed=3, dtype=dtype)
    clean = [torch.where(t.isfinite(), t, 0) for t in (ref.cache_values(cache[i], cache[2 + i]) for i in range(2))]
    for window, sees in ((None, True), (50, False)):
        got = layers.decode_attention(q.to(gpu), on[0], on[1], tables.to(gpu), torch.tensor(lengths, device=gpu),
                                      key_scales=on[2], value_scales=on[3], window=window).cpu()
        want, size = ref.attention(q, *clean, tables, lengths, window=window)
        p_step = 2.0 ** -16 if dtype == H16 and bits < 16 else half_step(dtype)
        bound = half_step(dtype) * want.abs() + (p_step + 2.0 ** -12) * size
        bad = torch.zeros(3, h, d, dtype=torch.bool)
        if sees:
            bad[0, :4, (slice(0, 32) if bits < 16 else slice(3, 4))] = True
        bad[1, 4:] = True
        assert not torch.isfinite(got[bad]).any()
        within(got[~bad], want[~bad], bound[~bad])


def test_attention_past_32_bit_offsets_and_late_positions(gpu):
    """Blocks whose offsets pass 2^31 bytes and elements, and rings near position 2^31."""
    g, block, d, few = 8, 64, 128, 6
    blocks = 2 ** 32 // (g * block * d) + few
    x, y = (rnd(few, g, block, d, seed=s) for s in (1, 2))
    small, big = (layers.quantized_cache(n, g, block, d, bits=8, device=gpu) for n in (few, blocks))
    slots = torch.arange(few * block, device=gpu)
    k, v = (t.transpose(1, 2).reshape(-1, g, d).to(gpu) for t in (x, y))
    layers.cache_write_quantized(k, v, slots, *small)
    layers.cache_write_quantized(k, v, slots + (blocks - few) * block, *big)
    for t, s in zip(big, small):
        t, s = (a[-few:].view(torch.uint8) for a in (t, s))
        same = bool((t == s).all())
        assert same
    for a, b in zip(layers.cache_read(slots, *small), layers.cache_read(slots + (blocks - few) * block, *big)):
        same = torch.equal(a, b)
        assert same
    q = rnd(2, 32, d, seed=3).to(gpu)
    tables = i32([[4, 0, 2], [5, 1, 3]], gpu)
    call = lambda c, t, lens, w=None: layers.decode_attention(  # noqa: E731
        q, c[0], c[1], t, torch.tensor(lens, device=gpu), key_scales=c[2], value_scales=c[3], window=w)
    assert torch.equal(call(big, tables + (blocks - few), [130, 192]), call(small, tables, [130, 192]))
    late = [2 ** 31 - 4096, 2 ** 31 - 5000]
    assert torch.equal(call(small, tables, late, 150), call(small, tables, [x - 192 * 11184000 for x in late], 150))


# --- norms and rotations --------------------------------------------------------------

def rope_case(dev, n, *, h=4, g=2, d=128, half=16, axes=1, sections=None, interleaved=False, dtype=B, far=1000, q_w=True,
              k_w=True, plus_one=True, eps=1e-6, seed=0, strided=False, i32s=False):
    q, k = rnd(n, h, d, seed=seed + 1, dtype=dtype), rnd(n, g, d, seed=seed + 2, dtype=dtype)
    ws = [rnd(d, seed=seed + s, dtype=dtype, std=0.3) if on else None for s, on in ((3, q_w), (4, k_w))]
    pos = torch.randint(0, far, (axes, n), generator=torch.Generator().manual_seed(seed))
    freq = (1.0 / (1e4 ** (torch.arange(half, dtype=torch.float32) / max(half, 1)))).float()
    qd, kd = q.to(dev), k.to(dev)
    if strided:
        wide = torch.full((n, h, 2 * d + 8), NAN, dtype=dtype, device=dev)
        wide[..., 8:8 + d] = qd
        qd = wide[..., 8:8 + d]
        kd = kd.transpose(0, 1).contiguous().transpose(0, 1)
    p = (pos[0] if axes == 1 else pos).to(torch.int32 if i32s else torch.int64)
    got = layers.qk_norm_rope(qd, kd, *(w if w is None else w.to(dev) for w in ws), p.to(dev), freq.to(dev), eps,
                              sections=sections, interleaved=interleaved, plus_one=plus_one)
    for x, w, y in zip((q, k), ws, got):
        assert y.is_contiguous()
        want, size = ref.norm_rope(x, w, pos.tolist(), freq.tolist(), eps, sections, interleaved, plus_one)
        within(y, want, half_step(dtype) * want.abs() + 2.0 ** -18 * size, (n, d, half))
    return got


@pytest.mark.parametrize("dtype", [B, H16])
@pytest.mark.parametrize("d,half", [(64, 8), (64, 32), (128, 16), (128, 48), (128, 64), (256, 32), (256, 128), (128, 0),
                                    (256, 96)])
def test_norm_rope_dims(gpu, dtype, d, half):
    for n in (1, 3, 33):
        rope_case(gpu, n, d=d, half=half, dtype=dtype, seed=n)


@pytest.mark.parametrize("axes,sections,interleaved", [(2, [10, 6], False), (3, [6, 5, 5], False), (3, [6, 5, 5], True),
                                                       (4, [4, 4, 4, 4], True), (3, [0, 16, 0], False),
                                                       (4, [10, 2, 1, 3], True), (1, [16], True), (1, [16], False)])
def test_norm_rope_axes(gpu, axes, sections, interleaved):
    rope_case(gpu, 19, axes=axes, sections=sections, interleaved=interleaved, seed=5, i32s=True)


@pytest.mark.parametrize("h,g", [(1, 1), (32, 8), (5, 3), (7, 7), (3, 0), (0, 3)])
def test_norm_rope_heads(gpu, h, g):
    rope_case(gpu, 9, h=h, g=g, seed=6)
    rope_case(gpu, 5, h=h, g=g, d=256, half=64, seed=6)


def test_norm_rope_strides_weights_and_options(gpu):
    rope_case(gpu, 17, strided=True, seed=7)
    rope_case(gpu, 1, strided=True, seed=7)
    rope_case(gpu, 17, q_w=False, seed=8)
    rope_case(gpu, 17, k_w=False, plus_one=False, eps=0.5, seed=9)
    rope_case(gpu, 17, q_w=False, k_w=False, d=64, half=32, seed=10)


def test_norm_rope_far_positions(gpu):
    """Angles of positions up to 2^31 - 1."""
    rope_case(gpu, 40, half=64, far=2 ** 31 - 1, seed=11, dtype=H16)
    rope_case(gpu, 40, half=64, axes=3, sections=[24, 20, 20], interleaved=True, far=1000000, seed=12)


def test_norm_rope_of_many_tokens(gpu):
    """A wave for all heads of a token gives what a wave for a few of them gives, bit for bit."""
    n = 5000
    q, k = rnd(n, 32, 128, seed=1).to(gpu), rnd(n, 8, 128, seed=2).to(gpu)
    w = [rnd(128, seed=s).to(gpu) for s in (3, 4)]
    pos, freq = torch.arange(n, device=gpu), torch.rand(32, generator=torch.Generator().manual_seed(5)).to(gpu)
    many = layers.qk_norm_rope(q, k, *w, pos, freq, 1e-6)
    for at in (0, 700, 4990):
        few = layers.qk_norm_rope(q[at:at + 10], k[at:at + 10], *w, pos[at:at + 10], freq, 1e-6)
        assert all(torch.equal(a, b[at:at + 10]) for a, b in zip(few, many))


# --- together ---------------------------------------------------------------------

class Decoder:
    """The layer that a user's program would have: tables, a quantised cache, and its steps."""

    def __init__(self, dev, requests, *, bits, h=8, g=2, d=128, block=16, columns=12, axes=1, seed=0):
        self.dev, self.h, self.g, self.d, self.block, self.bits = dev, h, g, d, block, bits
        self.cache = layers.quantized_cache(requests * columns, g, block, d, bits=bits, device=dev)
        self.tables = torch.full((requests, columns), -1, dtype=torch.int32, device=dev)
        self.free = torch.randperm(requests * columns, generator=torch.Generator().manual_seed(seed)).to(torch.int32).to(dev)
        self.count = i32([requests * columns], dev)
        self.w = [rnd(d, seed=seed + s, std=0.3).to(dev) for s in (1, 2)]
        self.freq = (1.0 / (1e4 ** (torch.arange(16, device=dev, dtype=torch.float32) / 16)))
        self.sections = None if axes == 1 else [6, 5, 5]

    def inputs(self, proj, positions):
        h, g, d = self.h, self.g, self.d
        n = proj.shape[0]
        qg = proj[:, :2 * h * d].view(n, h, 2 * d)
        k, v = (proj[:, 2 * h * d + i * g * d:][:, :g * d].view(n, g, d) for i in (0, 1))
        q, k = layers.qk_norm_rope(qg[..., :d], k, *self.w, positions, self.freq, 1e-6, sections=self.sections)
        return q, k, v, qg[..., d:]

    def write(self, k, v, lengths, cu, total):
        slots, _ = ik.extend_block_tables(lengths, cu, self.tables, self.free, self.count, self.block, total)
        layers.cache_write_quantized(k, v, slots, *self.cache)

    def step(self, proj, positions, lengths, cu, **kw):
        """One token a request behind lengths; returns the layer's read."""
        q, k, v, gate = self.inputs(proj, positions)
        self.write(k, v, lengths, cu, proj.shape[0])
        return layers.decode_attention(q, self.cache[0], self.cache[1], self.tables, lengths + 1,
                                       key_scales=self.cache[2], value_scales=self.cache[3], gate=gate, **kw)


@pytest.mark.parametrize("bits,axes", [(8, 1), (4, 3)])
def test_prefill_then_decode(gpu, bits, axes):
    """Prompts are written and decoded over; every read is the oracle's over the rows as quantised, and they read back."""
    prompts, steps, h, g, d = [37, 5, 90], 4, 8, 2, 128
    layer = Decoder(gpu, 3, bits=bits, axes=axes)
    rows = [[[], []] for _ in prompts]            # the oracle's keys and values of each request
    p_cu = torch.tensor([0] + prompts).cumsum(0)
    n = int(p_cu[-1])

    def record(q, k, v, cu):
        for r in range(3):
            for which, x in enumerate((k, v)):
                rows[r][which] += list(ref.quantise(x[cu[r]:cu[r + 1]].cpu(), bits)[0])
        return q.cpu()
    proj = rnd(n, 2 * h * d + 2 * g * d, seed=1).to(gpu)
    pos = torch.cat([torch.arange(x) for x in prompts])
    pos = torch.stack((pos, pos // 3, pos % 3)) if axes == 3 else pos
    q, k, v, _ = layer.inputs(proj, pos.to(gpu))
    record(q, k, v, p_cu.tolist())
    layer.write(k, v, torch.zeros(3, dtype=torch.int64, device=gpu), p_cu.to(gpu), n)
    lengths = torch.tensor(prompts, device=gpu)
    cu = torch.arange(4, device=gpu)
    slopes = torch.tensor([0.1 * i for i in range(h)], device=gpu)
    kw = dict(softcap=20.0, window=60, slopes=slopes)
    for step in range(steps):
        proj = rnd(3, 2 * h * d + 2 * g * d, seed=10 + step).to(gpu)
        pos = lengths if axes == 1 else torch.stack((lengths, lengths // 2, lengths % 5))
        got = layer.step(proj, pos, lengths, cu, **kw)
        q, k, v, gate = layer.inputs(proj, pos)
        q = record(q, k, v, range(4))
        lengths = lengths + 1
        for r, length in enumerate(lengths.tolist()):
            keys, values = (torch.stack(x).transpose(0, 1)[None] for x in rows[r])
            want, size = ref.attention(q[r:r + 1], keys, values, torch.zeros(1, 1, dtype=torch.int32), [length],
                                       gate=gate[r:r + 1].cpu(), softcap=20.0, window=60, slopes=slopes.cpu())
            within(got[r:r + 1], want, half_step(B) * want.abs() + (half_step(B) + 2.0 ** -12) * size, (step, r))
    total = int(lengths.sum())
    off = torch.cat((lengths.new_zeros(1), lengths.cumsum(0)))
    slots, _ = ik.slot_map(off, torch.zeros_like(lengths), layer.tables, layer.block, total)
    for which, x in enumerate(layers.cache_read(slots, *layer.cache)):
        want = torch.cat([torch.stack(rows[r][which]) for r in range(3)])
        assert torch.equal(x.cpu(), want.to(B))


@pytest.mark.parametrize("bits", [8, 4])
def test_captured_steps_and_padded_batches(gpu, bits):
    """A step captured for four rows, replayed with other inputs, lengths and idle rows, beside eager work."""
    layer = Decoder(gpu, 4, bits=bits, columns=100)
    h, g, d = layer.h, layer.g, layer.d
    prompts = torch.tensor([700, 0, 130, 1290], device=gpu)
    pc = torch.cat((prompts.new_zeros(1), prompts.cumsum(0)))
    n = int(pc[-1])
    k, v = (rnd(n, g, d, seed=s).to(gpu) for s in (1, 2))
    layer.write(k, v, torch.zeros_like(prompts), pc, n)
    proj, lengths = rnd(4, 2 * h * d + 2 * g * d, seed=3).to(gpu), prompts.clone()
    cu = torch.arange(5, device=gpu, dtype=torch.int32)

    def step():
        live = cu[1:] > cu[:-1]
        q, kk, vv, gate = layer.inputs(proj, lengths)
        slots, _ = ik.extend_block_tables(lengths, cu, layer.tables, layer.free, layer.count, 16, 4)
        layers.cache_write_quantized(kk, vv, slots, *layer.cache)
        seen = torch.where(live, lengths + 1, 0)
        return layers.decode_attention(q, layer.cache[0], layer.cache[1], layer.tables, seen,
                                       key_scales=layer.cache[2], value_scales=layer.cache[3], gate=gate, softcap=30.0)
    start = [x.clone() for x in (*layer.cache, layer.tables, layer.free, layer.count)]

    def reset():
        for x, y in zip((*layer.cache, layer.tables, layer.free, layer.count), start):
            x.copy_(y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    reset()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(step())
        reset()
    for turn in range(4):
        proj.copy_(rnd(4, 2 * h * d + 2 * g * d, seed=20 + turn).to(gpu))
        counts = [1, 1, 1, 1] if turn != 2 else [1, 0, 0, 1]
        cu.copy_(torch.tensor([0] + counts).cumsum(0))
        lengths.copy_(prompts + turn * 16)
        reset()
        want = step()
        state = [x.view(torch.uint8).clone() for x in layer.cache]
        assert bool((want[[i for i, c in enumerate(counts) if not c]] == 0).all())
        for graph, out in zip(graphs, outs):
            reset()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
            assert all(torch.equal(x.view(torch.uint8), y) for x, y in zip(layer.cache, state))


def test_two_streams_at_once(gpu):
    """Calls that overlap, each with its own scratch, give what they give alone."""
    x, y = (rnd(64, 2, 64, 64, seed=s) for s in (1, 2))
    c = [t.to(gpu) for t in cache_of(x, y, 8)]
    tables = i32([list(range(64))], gpu)
    qs = [rnd(1, 8, 64, seed=s).to(gpu) for s in (3, 4)]
    lens = [torch.tensor([n], device=gpu) for n in (4000, 3333)]
    call = lambda i: layers.decode_attention(qs[i], c[0], c[1], tables, lens[i], key_scales=c[2], value_scales=c[3])  # noqa: E731
    alone = [call(0), call(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(call(i))
    torch.cuda.synchronize()
    assert all(torch.equal(o, alone[i]) for i in range(2) for o in outs[i])


def test_unchanged_inputs_and_repeated_calls(gpu):
    """The same call gives the same bits, whatever ran between, and changes none of its inputs."""
    x, y = (rnd(40, 2, 16, 128, seed=s) for s in (1, 2))
    c = [t.to(gpu) for t in cache_of(x, y, 4)]
    q, tables, lens = rnd(2, 8, 128, seed=3).to(gpu), i32([list(range(20)), list(range(20, 40))], gpu), torch.tensor([320, 7], device=gpu)
    before = [t.view(torch.uint8).clone() for t in (*c, q.view(torch.uint8), tables.view(torch.uint8), lens.view(torch.uint8))]
    call = lambda: layers.decode_attention(q, c[0], c[1], tables, lens, key_scales=c[2], value_scales=c[3])  # noqa: E731
    first = call()
    torch.full((1 << 24,), NAN, device=gpu)
    assert torch.equal(first, call()) and math.isfinite(first.float().sum().item())
    after = [t.view(torch.uint8) for t in (*c, q.view(torch.uint8), tables.view(torch.uint8), lens.view(torch.uint8))]
    assert all(torch.equal(a, b) for a, b in zip(before, after))


def test_odd_arguments(gpu):
    """Vectors from the host or in int32, layers of one pool, broadcast gates, rows that are no rows, tables with room."""
    g, block, d, h, blocks = 2, 24, 64, 6, 10
    pool = [torch.zeros(3, *t.shape, dtype=torch.uint8, device=gpu) for t in layers.quantized_cache(blocks, g, block, d, device="cpu")]
    layer = [pool[0][1].view(torch.float8_e4m3fn), pool[1][1].view(torch.float8_e4m3fn), pool[2][1], pool[3][1]]
    n = 100
    k, v = (rnd(n, g, d, seed=s).to(gpu) for s in (1, 2))
    slots = torch.randperm(blocks * block, generator=torch.Generator().manual_seed(3))[:n]
    layers.cache_write_quantized(k, v, slots.to(torch.int32), *layer)                       # from the host
    assert not any(t[0].any() or t[2].any() for t in pool)
    spread = torch.zeros(n, 2, g, d, dtype=B, device=gpu)[:, 0]                             # rows of twice the width
    spread.copy_(k)
    again = [t.clone() for t in layer]
    layers.cache_write_quantized(spread, k.transpose(1, 2).contiguous().transpose(1, 2).copy_(v), slots.to(gpu), *again)
    for a, b in zip(layer, again):
        same = torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        assert same
    back = layers.cache_read(slots.to(torch.int32), *layer)
    for x, y in zip((k, v), back):
        same = torch.equal(y.cpu(), ref.quantise(x.cpu(), 8)[0].to(B))
        assert same
    q = rnd(2, h, d, seed=4).to(gpu)
    tables = i32([[3, 1, 0, 7], [9, 4, 5, 2]], gpu)
    gate = rnd(1, h, d, seed=5).to(gpu)
    lens = torch.tensor([70, 41])
    call = lambda q, tables, lens, gate, **kw: layers.decode_attention(  # noqa: E731
        q, layer[0], layer[1], tables, lens, key_scales=layer[2], value_scales=layer[3], gate=gate, **kw)
    plain = call(q, tables, lens.to(gpu), gate.expand(2, h, d).contiguous(), starts=torch.tensor([5, 0], device=gpu))
    wide = i32([[3, 1, 0, 7, -1, 50], [9, 4, 5, 2, 6, 8]], gpu)
    for got in (call(q, tables, lens, gate.expand(2, h, d), starts=torch.tensor([5, 0], dtype=torch.int32)),
                call(q.transpose(0, 1).contiguous().transpose(0, 1), wide[:, :4], lens.to(torch.int32), gate.expand(2, h, d),
                     starts=torch.tensor([5, 0])),
                call(q.repeat_interleave(2, 2)[..., ::2], wide, lens, gate.expand(2, h, d), starts=torch.tensor([5, 0]))):
        assert torch.equal(got, plain)
    one = call(q[:1], tables[:1], lens[:1], gate, starts=torch.tensor([5]))                 # a single row's strides say nothing
    assert torch.equal(one, plain[:1])
    x, pos = rnd(7, 3, 128, seed=6).to(gpu), torch.arange(21).view(7, 3).T
    freq = torch.rand(32, generator=torch.Generator().manual_seed(7))
    a = layers.qk_norm_rope(x, x, None, None, pos, freq[::2].to(gpu), 1e-6, sections=[6, 5, 5])
    b = layers.qk_norm_rope(x.expand(7, 3, 128), x[:, :1].expand(7, 3, 128), None, None, pos.to(gpu), freq[::2].contiguous().to(gpu),
                            1e-6, sections=(6, 5, 5))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1][:, :1].expand(7, 3, 128), b[1])


@pytest.mark.parametrize("bits,dtype", FORMS)
def test_idle_rows_may_hold_anything(gpu, bits, dtype):
    """Rows of a captured batch that no request has: queries, gates and tables of anything, zeros out; the others as ever."""
    x, y = (rnd(40, 2, 16, 64, seed=s, dtype=dtype) for s in (1, 2))
    c = [None if t is None else t.to(gpu) for t in (cache_of(x, y, bits) if bits < 16 else (x, y, None, None))]
    q, gate = rnd(4, 8, 64, seed=3, dtype=dtype).to(gpu), rnd(4, 8, 64, seed=4, dtype=dtype).to(gpu)
    tables, lens = torch.arange(160, dtype=torch.int32, device=gpu).view(4, 40) % 40, torch.tensor([600, 0, 30, 0], device=gpu)
    starts = torch.tensor([0, 0, 30, 5], device=gpu)
    call = lambda: layers.decode_attention(q, c[0], c[1], tables, lens, key_scales=c[2], value_scales=c[3], starts=starts, gate=gate)  # noqa: E731
    clean = call()
    q[1:] = NAN
    gate[1:] = torch.tensor([NAN, INF, -INF], device=gpu, dtype=dtype).view(3, 1, 1)
    tables[1:] = 1 << 30
    got = call()
    assert torch.equal(got[0], clean[0]) and not got[1:].any() and not clean[1:].any() and torch.isfinite(got).all()


def test_other_cuda_streams_own_scratch(gpu):
    """Inputs made on one stream, used on another that waits for it; scratch is the using stream's."""
    side = torch.cuda.Stream()
    x, y = (rnd(200, 1, 16, 128, seed=s) for s in (1, 2))
    c = [t.to(gpu) for t in cache_of(x, y, 4)]
    q, tables, lens = rnd(1, 4, 128, seed=3).to(gpu), i32([list(range(200))], gpu), torch.tensor([3200], device=gpu)
    want = layers.decode_attention(q, c[0], c[1], tables, lens, key_scales=c[2], value_scales=c[3])
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layers.decode_attention(q, c[0], c[1], tables, lens, key_scales=c[2], value_scales=c[3])
        rows = layers.cache_read(torch.arange(40, device=gpu), *c)
    torch.cuda.current_stream().wait_stream(side)
    noise = [torch.full((1 << 20,), NAN, device=gpu) for _ in range(4)]
    assert torch.equal(got, want) and rows[0].shape == (40, 1, 128) and len(noise) == 4


# --- what is not finite, in each value ------------------------------------------------

def same_or_within(got, want, bound, what=""):
    """As ``within`` where want is finite; elsewhere the same infinity, or NaN for NaN."""
    least = torch.finfo(got.dtype).smallest_normal * half_step(got.dtype) + 1e-30
    got, fine = got.detach().double().cpu(), want.isfinite()
    assert torch.equal(got[~fine].nan_to_num(7.0), want[~fine].nan_to_num(7.0)), (what, got[~fine], want[~fine])
    got[~fine] = 0
    zero = torch.zeros_like(want)
    bad = ~((got - torch.where(fine, want, zero)).abs() <= torch.where(fine, bound, zero) + least)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}"


def spoiled_case(dev, cache, lengths, h, dtype, d, block, seed, mark=None, **kw):
    """The case's output against the oracle over the cache as its product takes it (codes past bf16's range: infinities)."""
    r, blocks = len(lengths), cache[0].shape[0]
    columns = blocks // r
    tables = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed))[:r * columns].to(torch.int32).view(r, columns)
    cache = [None if t is None else t.clone() for t in cache]
    mark(cache, lambda i, p: (int(tables[i, p // block]), p % block))
    q = rnd(r, h, d, seed=seed + 3, dtype=dtype)
    full = [ref.cache_values(cache[i], cache[2 + i]) for i in range(2)]
    full = [t.to(B).double() if cache[2] is not None else t for t in full]
    on = [None if t is None else t.to(dev) for t in cache]
    got = layers.decode_attention(q.to(dev), on[0], on[1], tables.to(dev), torch.tensor(lengths, device=dev),
                                  key_scales=on[2], value_scales=on[3], **kw)
    want, _ = ref.attention(q, *full, tables, lengths, **kw)
    full[1] = full[1].nan_to_num(0.0, 0.0, 0.0)
    _, size = ref.attention(q, *full, tables, lengths, **kw)
    p_step = 2.0 ** -16 if dtype == H16 and cache[2] is not None else half_step(dtype)
    same_or_within(got, want, half_step(dtype) * want.abs() + (p_step + 2.0 ** -12) * size, (dtype, d, h, block))
    return got.cpu(), want


@pytest.mark.parametrize("dtype", [B, H16])
@pytest.mark.parametrize("d,h,block", [(64, 3, 16), (128, 4, 16), (128, 7, 16), (256, 4, 16), (128, 16, 16), (128, 20, 16),
                                       (256, 16, 24), (128, 4, 24), (64, 2, 1)])
def test_attention_nan_codes_stay_in_their_dim(gpu, dtype, d, h, block):
    """An e4m3 NaN in one value's dim is that dim's only, whatever lies beside it in a dword or a tile."""
    columns = -(-2100 // block)
    x, y = (rnd(3 * columns, 1, block, d, seed=s) for s in (1, 2))
    c = cache_of(x, y, 8)

    def mark(cache, at):
        for i, p, dim in ((0, 9, 3), (0, 30, 6), (1, 2000, d - 1), (1, 0, 8)):
            b, row = at(i, p)
            cache[1].view(torch.uint8)[b, 0, row, dim] = 0xff if dim == 3 else 0x7f
    got, _ = spoiled_case(gpu, c, [100, 2050, 700], h, dtype, d, block, 5, mark)
    assert got[0].isnan().sum() == 2 * h and got[1].isnan().sum() == 2 * h and got[2].isfinite().all()


@pytest.mark.parametrize("bits,huge", [(4, 3.0e38), (8, 3.31e38)])
@pytest.mark.parametrize("d,h,block", [(128, 4, 16), (64, 8, 16), (128, 16, 16), (256, 4, 24)])
def test_attention_values_that_round_past_bf16(gpu, bits, huge, d, h, block):
    """Rows whose largest value becomes 2^128: an infinity for its dim, and finite values beside it in the run."""
    columns = -(-200 // block)
    k, v = (rnd(200, 1, d, seed=s) for s in (1, 2))
    v[50, 0, 34], v[50, 0, 35], v[50, 0, 36] = huge, 9.0e37, -9.0e37
    v[70, 0, 9], v[70, 0, 8] = -huge, 9.0e37
    cache = layers.quantized_cache(2 * columns, 1, block, d, bits=bits, device=gpu)
    tables = torch.randperm(2 * columns, generator=torch.Generator().manual_seed(3)).to(torch.int32).view(2, columns)
    slots = torch.tensor([int(tables[0, p // block]) * block + p % block for p in range(200)])
    layers.cache_write_quantized(k.to(gpu), v.to(gpu), slots.to(gpu), *cache)
    val, s = ref.quantise(v, bits)
    assert s.max() == (253 if bits == 4 else 247) and val.max() == 2.0 ** 128
    q = rnd(2, h, d, seed=4)
    got = layers.decode_attention(q.to(gpu), cache[0], cache[1], tables.to(gpu), torch.tensor([200, 0], device=gpu),
                                  key_scales=cache[2], value_scales=cache[3])
    keys, values = (ref.quantise(t, bits)[0].transpose(0, 1)[None] for t in (k, v))
    values = values.to(B).double()
    one = torch.zeros(1, 1, dtype=torch.int32)
    want, _ = ref.attention(q[:1], keys, values, one, [200])
    _, size = ref.attention(q[:1], keys, values.nan_to_num(0.0, 0.0, 0.0), one, [200])
    assert want.isinf().sum() == 2 * h
    same_or_within(got[:1], want, half_step(B) * want.abs() + (half_step(B) + 2.0 ** -12) * size)
    assert not got[1].any()


@pytest.mark.parametrize("dtype", [B, H16])
@pytest.mark.parametrize("d,h,block", [(128, 4, 16), (64, 8, 16), (128, 7, 48), (256, 5, 16), (128, 16, 16), (64, 20, 16),
                                       (256, 3, 24), (128, 2, 1)])
def test_attention_infinite_values_are_infinite(gpu, dtype, d, h, block):
    """16-bit caches: an infinity gives an infinity, both signs NaN, in their dims alone, wherever they lie in a tile."""
    columns = -(-2100 // block)
    x, y = (rnd(3 * columns, 1, block, d, seed=s, dtype=dtype) for s in (1, 2))

    def mark(cache, at):
        for i, p, dim, z in ((0, 9, 3, INF), (0, 10, 5, -INF), (0, 20, 7, INF), (0, 22, 7, -INF), (0, 31, 9, NAN),
                             (0, 99, 10, INF), (1, 2049, 0, -INF), (1, 1, 1, INF), (1, 1000, 1, -INF)):
            b, row = at(i, p)
            cache[1][b, 0, row, dim] = z
    _, want = spoiled_case(gpu, [x, y, None, None], [100, 2050, 700], h, dtype, d, block, 5, mark)
    assert want[0].isinf().sum() == 3 * h and want[0].isnan().sum() == 2 * h and want[2].isfinite().all()
    _, want = spoiled_case(gpu, [x, y, None, None], [100, 2050, 700], h, dtype, d, block, 6, mark, window=60, softcap=9.0)
    assert want[0].isinf().sum() == h


@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("n", [300, 6000])
def test_attention_infinite_values_of_far_lower_scores(gpu, first, n):
    """An infinity whose weight float32 holds as zero beside the largest is still one, within a part and between parts."""
    d, h = 128, 4
    x, y = torch.zeros(n // 16 + 1, 1, 16, d, dtype=B), rnd(n // 16 + 1, 1, 16, d, seed=2)
    high, low = (n - 7, 3) if first else (3, n - 7)
    x[high // 16, 0, high % 16] = 5.0            # a score of 128 5 / sqrt(128) 4 = 226 over the others' zero
    y[low // 16, 0, low % 16, 17], y[low // 16, 0, low % 16, 18] = INF, -INF
    tables = torch.arange(n // 16 + 1, dtype=torch.int32)[None]
    q = torch.full((1, h, d), 4.0, dtype=B)
    got = layers.decode_attention(q.to(gpu), x.to(gpu), y.to(gpu), tables.to(gpu), torch.tensor([n], device=gpu))
    want, _ = ref.attention(q, x.double(), y.double(), tables, [n])
    _, size = ref.attention(q, x.double(), y.double().nan_to_num(0.0, 0.0, 0.0), tables, [n])
    assert want.isinf().sum() == 2 * h
    same_or_within(got, want, half_step(B) * want.abs() + (half_step(B) + 2.0 ** -12) * size)


@pytest.mark.parametrize("score,scale", [(2, 1), (13, 1024)])
@pytest.mark.parametrize("bits,dtype", FORMS)
def test_attention_of_equal_weights_beside_larger_ones(gpu, bits, dtype, score, scale):
    """Every 16th key has a score of 2 (13; 12 in 4 bits) and a value of 0, the others' weights are e^-2 (e^-13) of its,
    which a 16-bit type would round all the same way: by 2^-8.4 in bf16, 2^-11.7 in fp16 (2^-8.9, 2^-11.3).  The output
    is within half a step of its own binade and 2^-14 of sum p |v|: weights of two parts 2^-16, scores (exact, times
    log2(e) / 8 and less the largest: 2^-24 of 19 each) 2^-19, sums of at most 64 positions a lane and 100 parts 2^-17
    in numerator and denominator."""
    d, h, lengths = 64, 4, [18, 23, 29, 47, 64, 101, 333, 5000]
    blocks = 5008 // 16
    x, y = torch.zeros(blocks, 1, 16, d, dtype=dtype), torch.ones(blocks, 1, 16, d, dtype=dtype)
    x[:, 0, 3] = score / 8
    y[:] = (1 + torch.arange(d) / 64) * scale
    y[:, 0, 3] = 0
    cache = list(cache_of(x, y, bits)) if bits < 16 else [x, y, None, None]
    full = [ref.cache_values(cache[i], cache[2 + i]) for i in range(2)]
    tables = torch.arange(blocks, dtype=torch.int32).repeat(len(lengths), 1)
    q = torch.ones(len(lengths), h, d, dtype=dtype)
    on = [None if t is None else t.to(gpu) for t in cache]
    got = layers.decode_attention(q.to(gpu), on[0], on[1], tables.to(gpu), torch.tensor(lengths, device=gpu),
                                  key_scales=on[2], value_scales=on[3])
    want, size = ref.attention(q, *full, tables, lengths)
    step = torch.exp2(torch.floor(torch.log2(want * (1 + 2.0 ** -14)))) * half_step(dtype)
    within(got, want, step + 2.0 ** -14 * size, (bits, dtype))


@pytest.mark.parametrize("bits", [8, 4])
def test_read_every_scale_byte(gpu, bits):
    """All codes under each of the 256 scale bytes, those included that the write never makes."""
    codes = torch.arange(256).to(torch.uint8)
    d = 32 * len(codes.view(-1, 32 if bits == 8 else 16))
    keys = codes.view(1, 1, 1, -1).expand(256, 1, 1, -1).contiguous()
    s = torch.arange(256).to(torch.uint8).view(256, 1, 1, 1).expand(256, 1, d // 32, 1).contiguous()
    keys = keys.view(torch.float8_e4m3fn) if bits == 8 else keys
    for dtype in (B, H16):
        got = layers.cache_read(torch.arange(256, device=gpu), keys.to(gpu), keys.to(gpu), s.to(gpu), s.to(gpu), dtype=dtype)
        want = ref.cache_values(keys, s)[:, :, 0].to(dtype)
        for x in got:
            same = x.cpu() == want
            assert (same | (x.cpu().isnan() & want.isnan())).all(), (~same).nonzero()[:5].tolist()


# --- scratch that is used -----------------------------------------------------------

def scratch_case(dev, seed, lengths=(3200, 7)):
    """A call over 4 bits that needs its workspace, and the workspace's size."""
    r, g, block, d, h, columns = len(lengths), 2, 16, 128, 8, 200
    x, y = (rnd(r * columns, g, block, d, seed=seed + s) for s in (1, 2))
    c = [t.to(dev) for t in cache_of(x, y, 4)]
    q = rnd(r, h, d, seed=seed + 3).to(dev)
    tables = torch.arange(r * columns, dtype=torch.int32, device=dev).view(r, columns)
    lens = torch.tensor(lengths, device=dev)
    need = N.lib().yh_decode_attention_workspace_bytes(r, h, g, d, block, columns, 0, -1, 4, N.BF16)
    assert need > 0
    call = lambda: layers.decode_attention(q, c[0], c[1], tables, lens, key_scales=c[2], value_scales=c[3])  # noqa: E731
    return call, need, c


def test_scratch_of_earlier_calls_does_not_matter(gpu):
    """The memory that a call's scratch comes from is filled with NaN and with ones between calls: the same bits."""
    call, need, _ = scratch_case(gpu, 40)
    first = call()
    assert torch.isfinite(first).all() and first.any()
    for byte in (0xff, 0x00, 0x3f):
        torch.cuda.synchronize()
        dirt = [torch.full((need,), byte, dtype=torch.uint8, device=gpu) for _ in range(8)]
        where = {t.data_ptr() for t in dirt}
        del dirt
        again = torch.empty((need,), dtype=torch.uint8, device=gpu)
        assert again.data_ptr() in where       # the allocator gives what was just filled
        del again
        assert torch.equal(first, call())


def test_side_stream_work_beside_the_main_stream(gpu):
    """Calls queued on a side stream while the main stream allocates and fills memory of the scratch's size: each is right,
    as are rows read there."""
    call, need, c = scratch_case(gpu, 50)
    want, slots = call(), torch.arange(300, device=gpu)
    rows = layers.cache_read(slots, *c)
    for x, which in zip(rows, (0, 1)):
        full = ref.cache_values(c[which].cpu(), c[2 + which].cpu()).transpose(1, 2).reshape(-1, 2, 128)[:300]
        assert torch.equal(x.cpu(), full.to(B))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    busy = torch.randn(4096, 4096, device=gpu)
    outs, noise = [], []
    for _ in range(10):
        with torch.cuda.stream(side):
            busy @ busy                        # what follows is still queued when the noise starts
            outs.append((call(), layers.cache_read(slots, *c)))
        noise += [torch.full((need,), 0xff, dtype=torch.uint8, device=gpu) for _ in range(4)]
    assert not side.query()                    # there was work to run beside
    torch.cuda.current_stream().wait_stream(side)
    for got, back in outs:
        same = torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(back, rows))
        assert same


@pytest.mark.parametrize("bits,dtype", FORMS)
@pytest.mark.parametrize("block", [16, 24])
def test_attention_values_not_finite_beside_masks_biases_and_gates(gpu, bits, dtype, block):
    """Infinities (NaN codes over quantised caches) in seen positions, before starts, and in blocks taken out of the table,
    with caps, biases of both signs and gates; whole and in parts; replayed as a graph beside calls without such values."""
    d, g, h, lengths, starts = 128, 2, 8, [2100, 90, 300], [1000, 0, 40]
    columns = -(-2100 // block)
    x, y = (rnd(3 * columns, g, block, d, seed=s, dtype=dtype) for s in (1, 2))
    tables = torch.randperm(3 * columns, generator=torch.Generator().manual_seed(3)).to(torch.int32).view(3, columns)
    cache = list(cache_of(x, y, bits)) if bits < 16 else [x, y, None, None]
    clean = [None if t is None else t.clone() for t in cache]
    for i, p, dim in ((0, 999, 2), (0, 1000, 5), (0, 2099, 40), (1, 47, 7), (1, 89, 100), (2, 39, 1), (2, 200, 66)):
        b, row = int(tables[i, p // block]), p % block
        if bits == 16:
            cache[1][b, 1, row, dim] = -INF if dim == 5 else INF
        elif bits == 8:
            cache[1].view(torch.uint8)[b, 1, row, dim] = 0x7f
        else:
            cache[3][b, 1, dim // 32, row] = 255
    tables[1, 47 // block] = -1               # request 1 does not see position 47
    tables[2, 0] = 1 << 30
    q, gate = rnd(3, h, d, seed=4, dtype=dtype), rnd(3, h, d, seed=5, dtype=dtype)
    slopes = torch.tensor([0.01 * (i - 3) for i in range(h)])
    kw = dict(softcap=12.0, scale=0.1)
    full = [ref.cache_values(cache[i], cache[2 + i]) for i in range(2)]
    want, _ = ref.attention(q, *full, tables, lengths, starts=starts, slopes=slopes, gate=gate, **kw)
    full[1] = full[1].nan_to_num(0.0, 0.0, 0.0)
    _, size = ref.attention(q, *full, tables, lengths, starts=starts, slopes=slopes, gate=gate, **kw)
    assert want[:, :4].isfinite().all()       # those of the other KV head
    lost = 32 if bits == 4 else 1             # a scale is its run's
    assert [int((~want[i, 4:].isfinite()).sum()) for i in range(3)] == [4 * 2 * lost, 4 * lost, 4 * lost]
    on = [None if t is None else t.to(gpu) for t in cache]
    dq, dt, dl, ds = q.to(gpu), tables.to(gpu), torch.tensor(lengths, device=gpu), torch.tensor(starts, device=gpu)
    sl, dg = slopes.to(gpu), gate.to(gpu)
    call = lambda: layers.decode_attention(dq, on[0], on[1], dt, dl, key_scales=on[2], value_scales=on[3], starts=ds,  # noqa: E731
                                           slopes=sl, gate=dg, **kw)
    got = call()
    same_or_within(got, want, half_step(dtype) * want.abs() + (2.0 ** -16 + 2.0 ** -12) * size, (bits, dtype, block))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    spoiled = [None if t is None else t.clone() for t in on]
    for turn in range(3):
        for t, s, c in zip(on, spoiled, clean):
            if t is not None:
                t.view(torch.uint8).copy_((c.to(gpu) if turn == 1 else s).view(torch.uint8))
        eager = call()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.view(torch.int16), eager.view(torch.int16))
        assert torch.equal(eager.view(torch.int16), got.view(torch.int16)) == (turn != 1)
        assert eager.isfinite().all() == (turn == 1)
