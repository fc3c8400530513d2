"""Quantised caches without a GPU: the oracle's codes, what the wrappers and the C
calls refuse."""
import ctypes
import math

import pytest
import torch

from oracle import qcache as ref
from yanchor_amd import _native, layers

B, H16 = torch.bfloat16, torch.float16


def test_codes_are_the_types_own():
    e4m3 = torch.arange(256, dtype=torch.int32).to(torch.uint8).view(torch.float8_e4m3fn).double()
    assert torch.equal(ref.code_values(8).nan_to_num(9e9), e4m3.nan_to_num(9e9))
    assert ref.code_values(4).tolist() == [0, .5, 1, 1.5, 2, 3, 4, 6, -0.0, -.5, -1, -1.5, -2, -3, -4, -6]


@pytest.mark.parametrize("bits,most", [(8, 448.0), (4, 6.0)])
def test_no_value_saturates_and_scales_are_the_smallest(bits, most):
    gen = torch.Generator().manual_seed(bits)
    x = torch.randn(500, 64, generator=gen) * torch.exp2(torch.randint(-40, 40, (500, 1), generator=gen).float())
    x[0, :32] = 0
    x[1, 3], x[2, 40], x[3, 5] = math.inf, math.nan, most * 4
    val, s = ref.quantise(x, bits)
    assert s[0, 0] == 16 and s[1, 0] == 255 and s[1, 1] < 255 and s[2, 1] == 255
    runs, got = x.double().view(500, 2, 32), val.view(500, 2, 32)
    top = runs.abs().amax(-1)
    fine = s < 255
    unit = 2.0 ** (s.double() - 127)
    assert (top[fine] <= most * unit[fine]).all() and (top[fine & (s > 16)] > most * unit[fine & (s > 16)] / 2).all()
    # half a step: of e4m3 2^-4 of the value, of e2m1 a quarter of its power of two; near zero half the smallest code
    least = {8: 2.0 ** -10, 4: 0.25}[bits] * unit[..., None]
    step = {8: 2.0 ** -4, 4: 0.25}[bits] * runs.abs()
    assert (((runs - got).abs() <= torch.maximum(step, least))[fine]).all()
    assert got[~fine].isnan().all()
    assert ref.quantise(torch.full((1, 32), most), bits)[1].item() == 127
    assert ref.quantise(torch.full((1, 32), most * (1 + 2.0 ** -8)), bits)[1].item() == 128


def test_oracle_attention_of_a_full_table_is_softmax_attention():
    torch.manual_seed(2)
    q = torch.randn(1, 4, 64)
    keys, values = torch.randn(3, 2, 8, 64).double(), torch.randn(3, 2, 8, 64).double()
    out, _ = ref.attention(q, keys, values, torch.tensor([[2, 0, 1]]), [20])
    k = keys[[2, 0, 1]].transpose(1, 2).reshape(24, 2, 64)[:20].repeat_interleave(2, 1)
    v = values[[2, 0, 1]].transpose(1, 2).reshape(24, 2, 64)[:20].repeat_interleave(2, 1)
    want = torch.nn.functional.scaled_dot_product_attention(q.double().transpose(0, 1), k.transpose(0, 1), v.transpose(0, 1))
    assert torch.allclose(out[0], want[:, 0], rtol=1e-12, atol=1e-12)


# --- refusals: nothing reaches a device ---------------------------------------

def cache8(blocks=2, g=2, block=16, d=128):
    return layers.quantized_cache(blocks, g, block, d, bits=8, device="cpu")


def test_quantized_cache_forms():
    k, v, ks, vs = cache8(3, 2, 16, 96)
    assert k.shape == v.shape == (3, 2, 16, 96) and k.dtype == torch.float8_e4m3fn
    assert ks.shape == vs.shape == (3, 2, 3, 16) and ks.dtype == torch.uint8 and not ks.any()
    k, _, ks, _ = layers.quantized_cache(1, 1, 1, 64, bits=4, device="cpu")
    assert k.shape == (1, 1, 1, 32) and k.dtype == torch.uint8 and ks.shape == (1, 1, 2, 1)
    for kw in (dict(bits=16), dict(dim=48), dict(dim=0), dict(groups=0), dict(block=0), dict(blocks=-1)):
        a = dict(blocks=1, groups=1, block=16, dim=64, bits=8)
        a.update(kw)
        with pytest.raises(ValueError):
            layers.quantized_cache(a["blocks"], a["groups"], a["block"], a["dim"], bits=a["bits"], device="cpu")


def test_write_and_read_refuse():
    c = cache8()
    x, one = torch.zeros(3, 2, 128, dtype=B), torch.zeros(3, dtype=torch.int64)
    for k, v, cache, match in [
        (x.float(), x.float(), c, "bf16 / fp16"), (x, x[:2], c, "bf16 / fp16"), (x[:, :1], x[:, :1], c, "8-bit cache"),
        (x, x, (c[0], c[1], c[2][:1], c[3]), "scales"), (x, x, (c[0], c[1], None, None), "scales"),
        (x, x, (c[0].view(torch.uint8), c[1].view(torch.uint8), c[2], c[3]), "4-bit cache"),
        (x, x, (c[0].transpose(1, 2), c[1].transpose(1, 2), c[2], c[3]), "contiguous"),
        (x, x, (c[0].float(), c[1].float(), c[2], c[3]), "bf16, fp16"), (x, x, c, "ROCm device"),
    ]:
        with pytest.raises(ValueError, match=match):
            layers.cache_write_quantized(k, v, one, *cache)
    half = torch.zeros(2, 2, 16, 128, dtype=B)
    for args, kw, match in [
        ((half, half), dict(dtype=H16), "16-bit cache must be"), ((half, half, c[2], c[3]), {}, "no scales"),
        (c, dict(dtype=torch.float32), "bf16 or fp16"), (c, {}, "ROCm device"), ((half[0], half[0]), {}, "contiguous"),
        ((half[..., :4].contiguous(),) * 2, {}, "16 bytes"),
    ]:
        with pytest.raises(ValueError, match=match):
            layers.cache_read(one, *args, **kw)


@pytest.mark.parametrize("kw,match", [
    (dict(q=torch.zeros(2, 8, 128)), "bf16 / fp16"),
    (dict(q=torch.zeros(2, 7, 128, dtype=B)), "dividing"),
    (dict(q=torch.zeros(2, 8, 96, dtype=B)), "64, 128 or 256"),
    (dict(q=torch.zeros(2, 8, 64, dtype=B)), "8-bit cache"),
    (dict(key_scales=None), "scales"),
    (dict(block_tables=torch.zeros(1, 2, dtype=torch.int32)), "block_tables"),
    (dict(block_tables=torch.zeros(2, 2, dtype=torch.int64)), "block_tables"),
    (dict(window=0), "window"), (dict(scale=0.0), "scale"), (dict(scale=math.nan), "scale"),
    (dict(softcap=0.0), "softcap"), (dict(softcap=-3.0), "softcap"), (dict(softcap=math.inf), "softcap"),
    (dict(slopes=torch.zeros(2)), "slopes"), (dict(slopes=torch.zeros(8, dtype=B)), "slopes"),
    (dict(gate=torch.zeros(2, 8, 64, dtype=B)), "gate"), (dict(lengths=torch.zeros(3, dtype=torch.int64)), "2 entries"),
    (dict(lengths=torch.zeros(2)), "integer"), (dict(starts=torch.zeros(1, dtype=torch.int64)), "2 entries"),
    (dict(), "ROCm device"),
])
def test_attention_refuses(monkeypatch, kw, match):
    if match != "ROCm device":      # what is checked behind the device
        monkeypatch.setattr(layers._tree, "device_of", lambda *a: torch.device("cpu"))
    k, v, ks, vs = cache8()
    a = dict(q=torch.zeros(2, 8, 128, dtype=B), keys=k, values=v, block_tables=torch.zeros(2, 2, dtype=torch.int32),
             lengths=torch.tensor([3, 9]), key_scales=ks, value_scales=vs)
    a.update(kw)
    with pytest.raises(ValueError, match=match):
        layers.decode_attention(**a)


@pytest.mark.parametrize("kw,match", [
    (dict(q=torch.zeros(3, 2, 96, dtype=B), k=torch.zeros(3, 1, 96, dtype=B)), "64, 128 or 256"),
    (dict(k=torch.zeros(3, 1, 64, dtype=B)), "one dtype"), (dict(k=torch.zeros(3, 1, 128, dtype=H16)), "one dtype"),
    (dict(q_w=torch.zeros(64, dtype=B)), "weights"), (dict(k_w=torch.zeros(128)), "weights"),
    (dict(inv_freq=torch.ones(12)), "inv_freq"), (dict(inv_freq=torch.ones(72)), "inv_freq"),
    (dict(inv_freq=torch.ones(16, dtype=B)), "inv_freq"), (dict(eps=-1.0), "eps"), (dict(eps=math.nan), "eps"),
    (dict(positions=torch.zeros(4, dtype=torch.int64)), "positions"), (dict(positions=torch.zeros(3)), "positions"),
    (dict(positions=torch.zeros(5, 3, dtype=torch.int64)), "positions"),
    (dict(positions=torch.zeros(2, 3, dtype=torch.int64)), "sections"),
    (dict(positions=torch.zeros(2, 3, dtype=torch.int64), sections=[8, 7]), "sections"),
    (dict(positions=torch.zeros(2, 3, dtype=torch.int64), sections=[17, -1]), "sections"),
    (dict(positions=torch.zeros(3, 3, dtype=torch.int64), sections=[8, 8]), "sections"),
    (dict(positions=torch.zeros(2, 3, dtype=torch.int64), sections=[7, 9], interleaved=True), "past the pairs"),
    (dict(), "ROCm device"),
])
def test_norm_rope_refuses(kw, match):
    a = dict(q=torch.zeros(3, 2, 128, dtype=B), k=torch.zeros(3, 1, 128, dtype=B), q_w=None, k_w=None,
             positions=torch.zeros(3, dtype=torch.int64), inv_freq=torch.ones(16), eps=1e-6)
    a.update(kw)
    with pytest.raises(ValueError, match=match):
        layers.qk_norm_rope(**a)


@pytest.fixture(scope="module")
def lib():
    return _native.lib()


def test_c_calls_refuse_before_device_work(lib):
    p, odd = ctypes.c_void_p(256), ctypes.c_void_p(264)

    def refused(rc, text):
        assert rc == -1 and text in lib.yh_last_error(), (rc, lib.yh_last_error())

    def write(k=p, ks=256, n=4, blocks=2, g=2, d=128, block=16, bits=8, dtype=1, scales=p, keys=p):
        return lib.yh_cache_write_quantized(k, ks, p, 256, p, keys, p, scales, p, n, blocks, g, d, block, bits, dtype, None)
    refused(write(bits=16), b"4 or 8")
    refused(write(dtype=0), b"bf16 or f16")
    refused(write(d=48), b"multiple of 32")
    refused(write(scales=None), b"null")
    refused(write(k=odd), b"aligned")
    refused(write(keys=odd), b"aligned")
    refused(write(ks=128), b"whole heads")
    refused(write(block=0), b"bad sizes")
    refused(write(n=(1 << 31) - 1), b"too large")
    assert write(n=0) == 0 and write(blocks=0, keys=None, scales=None) == 0

    def read(k=p, n=4, blocks=2, d=128, bits=8, dtype=1, scales=p):
        return lib.yh_cache_read(p, p, p, scales, scales, k, p, n, blocks, 2, d, 16, bits, dtype, None)
    refused(read(bits=5), b"4, 8 or 16")
    refused(read(dtype=0), b"bf16 or f16")
    refused(read(d=12, bits=16), b"multiple of 8")
    refused(read(scales=None), b"null")
    refused(read(k=odd), b"aligned")
    refused(read(k=None), b"null")
    assert read(n=0) == 0

    def attn(q=p, qs=1024, lengths=p, scales=p, gate=None, ghs=0, blocks=2, columns=2, h=8, g=2, d=128, block=16,
             window=0, scale=1.0, cap=0.0, bits=8, dtype=1, ws=1 << 30, n=1):
        return lib.yh_decode_attention(q, qs, p, p, scales, scales, p, lengths, None, None, gate, 1024, ghs, p, n, blocks,
                                       columns, h, g, d, block, window, -1, scale, cap, bits, dtype, p, ws, None)
    refused(attn(d=96), b"64, 128 or 256")
    refused(attn(h=7), b"bad sizes")
    refused(attn(columns=0), b"bad sizes")
    refused(attn(window=-1), b"bad sizes")
    refused(attn(bits=7), b"4, 8 or 16")
    refused(attn(scale=0.0), b"scale")
    refused(attn(cap=-1.0), b"softcap")
    refused(attn(cap=math.nan), b"softcap")
    refused(attn(lengths=None), b"null")
    refused(attn(scales=None), b"scales")
    refused(attn(scales=odd), b"aligned")
    refused(attn(q=odd), b"aligned")
    refused(attn(qs=512), b"whole heads")
    refused(attn(gate=p, ghs=64), b"gate strides")
    refused(attn(n=1 << 20), b"too large")
    refused(attn(n=1 << 15, columns=1 << 26), b"too large")
    need = lib.yh_decode_attention_workspace_bytes(1, 8, 2, 128, 16, 900, 0, -1, 8, 1)
    assert need > 0 and lib.yh_decode_attention_workspace_bytes(1, 8, 2, 128, 16, 900, 100, -1, 8, 1) == 0
    refused(attn(columns=900, ws=need - 1), b"workspace")
    assert attn(dtype=0) == -3 and attn(n=0) == 0

    def rope(q=p, d=128, rotary=32, axes=1, sections=None, interleaved=0, n=4, h=2, g=1, dtype=1, qts=256, eps=1e-6, pos=p):
        sec = None if sections is None else (ctypes.c_int64 * len(sections))(*sections)
        return lib.yh_qk_norm_rope(q, qts, 128, p, 128, 128, p, p, pos, p, sec, axes, interleaved, p, p, n, h, g, d, rotary,
                                   eps, 1, dtype, None)
    refused(rope(d=96), b"64, 128 or 256")
    refused(rope(rotary=24), b"multiple of 16")
    refused(rope(rotary=144), b"multiple of 16")
    refused(rope(axes=5), b"axes")
    refused(rope(axes=2), b"sections")
    refused(rope(axes=2, sections=[8, 9]), b"add up")
    refused(rope(axes=2, sections=[17, -1]), b"bad section")
    refused(rope(axes=2, sections=[7, 9], interleaved=1), b"past the pairs")
    refused(rope(q=odd), b"aligned")
    refused(rope(q=None), b"null")
    refused(rope(pos=None), b"null")
    refused(rope(qts=12), b"aligned")
    refused(rope(eps=math.nan), b"eps")
    assert rope(dtype=0) == -3 and rope(n=0) == 0


@pytest.mark.parametrize("d,block", [(128, 1 << 30), (256, 1 << 29), (256, 613566757), (256, (1 << 31) - 16)])
@pytest.mark.parametrize("bits", [4, 8])
def test_attention_refuses_blocks_whose_scales_pass_32_bits(lib, d, block, bits):
    """A block's scales of one head are D / 32 runs of ``block`` bytes, which the kernel counts in 32 bits."""
    p = ctypes.c_void_p(256)
    rc = lib.yh_decode_attention(p, 8 * d, p, p, p, p, p, p, None, None, None, 0, 0, p, 1, 1, 1, 8, 2, d, block, 0, -1, 1.0, 0.0,
                                 bits, 1, p, 1 << 40, None)
    assert rc == -1 and b"too large" in lib.yh_last_error(), (rc, lib.yh_last_error())


def test_write_of_a_16_bit_cache_names_what_it_takes():
    half, x = torch.zeros(2, 2, 16, 128, dtype=B), torch.zeros(3, 2, 128, dtype=B)
    scales = cache8()[2:]
    for args in ((half, half, None, None), (half, half, *scales)):
        with pytest.raises(ValueError, match="4 or 8 bits"):
            layers.cache_write_quantized(x, x, torch.zeros(3, dtype=torch.int64), *args)
