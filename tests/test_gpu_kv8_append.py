"""Scales, gaps and ties of the append to 8-bit pages, beside tests/test_gpu_kv8.py."""
import math

import numpy as np
import pytest
import torch

import jitllm_b200 as jl
from jitllm_b200 import GGMLType
from tests import kv8_ref as ref
from tests.test_gpu_kv8 import _Pages, _stream, _up

pytestmark = pytest.mark.gpu


def _append(p, k, v, slot_map, positions=None, cos=None, sin=None, f16=False):
    keep = [_up(k), _up(v), _up(slot_map)]
    rope = {}
    if cos is not None:
        keep += [_up(positions), _up(cos), _up(sin)]
        rope = dict(positions=keep[3].data_ptr(), ropeCos=keep[4].data_ptr(), ropeSin=keep[5].data_ptr(), ropeRows=len(cos))
    jl.Kv8Append(p.pages, keep[0].data_ptr(), keep[1].data_ptr(), GGMLType.F16 if f16 else GGMLType.F32, tokens=len(slot_map), slotMap=keep[2].data_ptr(),
                 **rope).launch(_stream())
    torch.cuda.synchronize()


@pytest.mark.parametrize("d,heads", [(64, 5), (96, 3), (128, 8), (192, 2), (256, 1)])
@pytest.mark.parametrize("rope", [False, True])
@pytest.mark.parametrize("f16", [False, True])
def test_scales_are_rounded_once(dev, d, heads, rope, f16):
    """A scale is the binary32 number nearest to the largest element over 127. Of a rotated key that element is one of binary32: its products and
    their sum are off by (1 + sqrt 2) 2^-24 of it (no element of a pair is above sqrt 2 times the larger of the rotated two), the scale
    by 2^-24 more."""
    rng = np.random.default_rng(d)
    tokens, block = 2000, 16
    p = _Pages(dev, tokens // block, block, heads, d)
    codes, scales = p.host()
    dtype = np.float16 if f16 else np.float32
    k, v = ((rng.standard_normal((tokens, heads, d)) * np.exp(rng.standard_normal((tokens, heads, 1)))).astype(dtype) for _ in range(2))
    k[::7] = np.sign(k[::7]) * np.abs(k[::7, :, :1])  # rows whose elements are all as large
    slot_map, positions = rng.permutation(tokens).astype(np.int64), rng.integers(0, 4000, tokens).astype(np.int32)
    positions[:50] = 0
    cos, sin = ref.rope_tables(4000, d)
    ref.append_ref(codes, scales, k, v, slot_map, tokens, positions, cos if rope else None, sin)
    _append(p, k, v, slot_map, positions, cos if rope else None, sin, f16)
    got_codes, got_scales = p.host()
    assert np.array_equal(got_codes, codes)
    assert np.array_equal(got_scales[1].astype(np.float32), scales[1].astype(np.float32))
    if rope:
        assert (np.abs(got_scales[0] - scales[0]) <= (2 + math.sqrt(2)) * 2.0 ** -24 * scales[0]).all()
    else:
        assert np.array_equal(got_scales[0].astype(np.float32), scales[0].astype(np.float32))


def test_scales_of_every_size_are_rounded_once(dev):
    """Largest elements over all exponents from the one that is stored as zero to the largest, each with the fractions next to which a quotient by 127
    lies nearest to the middle of two numbers."""
    d, heads, block = 64, 4, 16
    fractions = np.concatenate((np.arange(8), 2 ** 23 - 1 - np.arange(8), np.random.default_rng(2).integers(0, 2 ** 23, 16))).astype(np.int64)
    bits = ((np.arange(26, 255)[:, None] << 23) | fractions[None]).astype(np.uint32).reshape(-1)
    most = np.resize(bits, -(-len(bits) // (heads * block)) * heads * block).view(np.float32)
    tokens = len(most) // heads
    rng = np.random.default_rng(3)
    p = _Pages(dev, tokens // block, block, heads, d)
    codes, scales = p.host()
    x = most.reshape(tokens, heads, 1) * rng.uniform(-0.99, 0.99, (tokens, heads, d)).astype(np.float32)
    x[:, :, 11] = most.reshape(tokens, heads)
    slot_map = np.arange(tokens, dtype=np.int64)
    ref.append_ref(codes, scales, x, -x, slot_map, tokens)
    _append(p, x, -x, slot_map)
    got_codes, got_scales = p.host()
    assert np.array_equal(got_codes, codes) and np.array_equal(got_scales.astype(np.float32), scales.astype(np.float32))


@pytest.mark.parametrize("d,heads,block,tokens,gap", [(64, 2, 16, 1, 0), (96, 3, 5, 33, 1), (128, 8, 16, 300, 2), (192, 2, 32, 65, 3), (256, 1, 16, 40, 5), (128, 5, 64, 700, 7)])
def test_append_writes_its_places_and_nothing_else(dev, d, heads, block, tokens, gap):
    """All memory of codes and of scales, between blocks and behind them too, bit for bit."""
    rng = np.random.default_rng(tokens)
    p = _Pages(dev, -(-tokens // block) + 3, block, heads, d, seed=tokens, gap=gap)
    want, want_scales = p.raw.clone(), p.raw_scales.clone()
    codes, scales = p.host()
    k, v = (rng.standard_normal((tokens, heads, d)).astype(np.float32) for _ in range(2))
    slot_map = rng.permutation(p.shape[0] * block)[:tokens].astype(np.int64)
    slot_map[:tokens // 4] = -1
    ref.append_ref(codes, scales, k, v, slot_map, tokens)
    want.as_strided(p.codes.shape, p.codes.stride(), p.codes.storage_offset()).copy_(_up(codes))
    want_scales.as_strided(p.scales.shape, p.scales.stride(), p.scales.storage_offset()).copy_(_up(scales.astype(np.float32)))
    _append(p, k, v, slot_map)
    assert torch.equal(p.raw, want) and torch.equal(p.raw_scales, want_scales)


@pytest.mark.parametrize("count", [0, -5, -2 ** 31])
def test_append_of_no_tokens_writes_nothing(dev, count):
    p = _Pages(dev, 4, 16, 2, 128, seed=3)
    codes, scales = p.raw.clone(), p.raw_scales.clone()
    k, m, n = torch.ones((8, 2, 128), device="cuda"), torch.arange(8, device="cuda"), torch.tensor([count], dtype=torch.int32, device="cuda")
    jl.Kv8Append(p.pages, k.data_ptr(), k.data_ptr(), GGMLType.F32, tokens=8, slotMap=m.data_ptr(), tokenCount=n.data_ptr()).launch(_stream())
    torch.cuda.synchronize()
    assert torch.equal(p.raw, codes) and torch.equal(p.raw_scales, scales)
