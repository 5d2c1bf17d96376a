"""What the attention over 8-bit pages keeps of tokens that weigh little: outputs element by element against 64 bits, relative to the
sum of their terms' magnitudes, where a token far above the others has nothing to say about an element."""
import math

import numpy as np
import pytest
import torch

import jitllm_b200 as jl
from tests.test_gpu_kv8 import _Attention, _stream

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ws(dev):
    w = jl.Kv8Workspace(dev)
    yield w
    w.close()


def _terms(a, r, h):
    """Row r, query head h in 64 bits: scores [tokens], outputs and the sums of their terms' magnitudes [size]; and of those terms whose weight
    times scale is below 2^-120 of the largest one: exponentials end at 2^-126 of it, in front of a scale of up to 2^4."""
    codes, scales = a.p.host()
    n = int(a.positions[r]) + 1
    j = np.arange(n)
    slot = r if a.kv_slots is None else int(a.kv_slots[r])
    b = a.table[slot][j // a.block]
    kv = h // (a.heads // codes.shape[2])
    k, v = (codes[w, b, kv, j % a.block].astype(np.float64) * scales[w, b, kv, j % a.block].astype(np.float64)[:, None] for w in (0, 1))
    s = k @ a.q[r, h * a.d:(h + 1) * a.d].astype(np.float64) * a.scale
    p = np.exp(s - s.max())
    p /= p.sum()
    weight = p * scales[1, b, kv, j % a.block]
    return s, p @ v, p @ np.abs(v), np.where(weight < 2.0 ** -120 * weight.max(), p, 0) @ np.abs(v)


def _tolerance(s, v_octaves, steps):
    """Of an output, relative to the sum of its terms' magnitudes. With X the largest |score| and G the widest distance of two
    scores in octaves (v_octaves: of two scales of values; 5: how far a weight may grow in front of a new reference), a weight is off by
    the score's five roundings and the subtraction's (2^-24 (5 X + G + v_octaves + 5) ln 2), the exponential (2^-22), the product with its
    scale (2^-24) and the digits that it is cut into (2^-18); the same but the last two again in the denominator. Weights of less than
    2^-41 of the largest may lose 2^-13 of an output together. Sums of `steps` steps of a warp in numerator (three additions each) and
    denominator (four), and 64 roundings of the warps' and parts' joins and the division."""
    x, g = np.abs(s).max() / math.log(2), (s.max() - s.min()) / math.log(2) + v_octaves
    return 2 * math.log(2) * 2.0 ** -24 * (5 * x + g + 5) + 2 * 2.0 ** -22 + 2.0 ** -24 + 2.0 ** -18 + (2.0 ** -13 if g >= 41 else 0) + (7 * steps + 64) * 2.0 ** -24


def _check_elements(a, v_octaves, steps, rows=None):
    torch.cuda.synchronize()
    got = a.out.cpu().numpy().astype(np.float64)
    worst = 0.0
    for r in range(a.rows) if rows is None else rows:
        for h in range(a.heads):
            s, want, size, beyond = _terms(a, r, h)
            far = np.abs(got[r, h * a.d:(h + 1) * a.d] - want)
            tol = _tolerance(s, v_octaves, steps) * size + beyond + 2.0 ** -149
            assert (far <= tol).all(), (r, h, float(np.max(far / np.maximum(size, 1e-300))), float(_tolerance(s, v_octaves, steps)), float(size.max()))
            worst = max(worst, float(np.max(far / np.maximum(size, 1e-300))))
    return worst


def _set_token(a, r, token, which, codes, scale):
    """Codes [kv heads or 1, size] and scale of a token of row r."""
    slot = r if a.kv_slots is None else int(a.kv_slots[r])
    b, at = int(a.table[slot, token // a.block]), token % a.block
    a.p.codes[which, b, :, at] = torch.as_tensor(np.broadcast_to(codes, (a.p.codes.shape[2], a.d)).astype(np.int8)).cuda()
    a.p.scales[which, b, :, at] = float(scale)


def _even_pages(a, key_scale, value_scale=0.01):
    """Scores of about one nat around 0, values above 0 everywhere."""
    rng = np.random.default_rng(7)
    shape = tuple(a.p.codes.shape[1:])
    a.p.codes[0] = torch.from_numpy(np.clip(np.rint(rng.standard_normal(shape) * 45), -127, 127).astype(np.int8)).cuda()
    a.p.codes[1] = torch.from_numpy(np.clip(np.rint(np.abs(rng.standard_normal(shape)) * 45) + 5, 1, 127).astype(np.int8)).cuda()
    a.p.scales[0] = key_scale
    a.p.scales[1] = value_scale
    q = np.abs(rng.standard_normal((a.rows, a.heads, a.d))) * 0.3 + 0.3
    q *= a.d * 0.5 / q.sum(-1, keepdims=True)  # every head's query has the same sum
    a.q[:, :a.heads * a.d] = q.reshape(a.rows, -1)
    a.dq.copy_(torch.from_numpy(a.q))


HEADS = [(64, 4, 1), (64, 8, 1), (96, 4, 2), (96, 16, 2), (128, 8, 2), (128, 6, 1), (192, 2, 2), (256, 4, 1)]


@pytest.mark.parametrize("d,heads,kv_heads", HEADS)
@pytest.mark.parametrize("gap", [6.0, 12.0, 16.0, 20.0, 40.0, 80.0])
def test_tokens_far_below_the_largest_keep_their_part(dev, ws, d, heads, kv_heads, gap):
    """One token is e^gap above the others and has zeros in every second element, which the others alone make up."""
    n, block = 700, 16
    for at in (0, 333):
        a = _Attention(dev, ws, rows=1, heads=heads, kv_heads=kv_heads, d=d, block=block, lengths=[n], own_slots=True, unwritten=False, seed=d + heads)
        _even_pages(a, 1 / (45 * 0.55))
        _set_token(a, 0, at, 0, 100, gap / (100 * d * 0.5 * a.scale))
        _set_token(a, 0, at, 1, np.where(np.arange(d) % 2, 0, 100), 0.01)
        for h in range(heads):
            s = _terms(a, 0, h)[0]
            assert abs(s[at] - gap) < 1e-3 and np.abs(np.delete(s, at)).max() < 5
        a.call().launch(_stream())
        _check_elements(a, 0, 8)


def test_tokens_far_below_the_largest_in_pages_of_odd_blocks_and_binary16(dev, ws):
    for f16, gap in ((False, 25.0), (True, 9.0)):
        a = _Attention(dev, ws, rows=3, heads=8, kv_heads=2, d=128, block=5, lengths=[31, 200, 1500], f16=f16, own_slots=True, unwritten=False, seed=2)
        _even_pages(a, 1 / (45 * 0.55))
        for r in range(3):
            _set_token(a, r, 17, 0, 100, gap / (100 * 64 * a.scale))
            _set_token(a, r, 17, 1, np.where(np.arange(128) % 2, 0, 100), 0.01)
        a.call().launch(_stream())
        torch.cuda.synchronize()
        if not f16:
            _check_elements(a, 0, 12)
            continue
        got = a.out.float().cpu().numpy().astype(np.float64)
        for r in range(3):
            for h in range(8):
                s, want, size, _ = _terms(a, r, h)
                far = np.abs(got[r, h * 128:(h + 1) * 128] - want)  # binary16 rounds each output by 2^-11 of it, or 2^-25
                assert (far <= (_tolerance(s, 0, 12) + 2.0 ** -11) * size + 2.0 ** -25).all()


@pytest.mark.parametrize("octaves", [10, 14, 20, 28, 60, 100])
@pytest.mark.parametrize("d,heads,kv_heads", [(64, 4, 1), (128, 8, 2), (128, 8, 1), (256, 2, 1)])
def test_a_value_with_a_large_scale_and_one_code_leaves_the_other_elements(dev, ws, octaves, d, heads, kv_heads):
    a = _Attention(dev, ws, rows=1, heads=heads, kv_heads=kv_heads, d=d, block=16, lengths=[750], own_slots=True, unwritten=False, seed=3)
    _even_pages(a, 1 / (45 * 0.55))
    only = np.zeros(d)
    only[5] = 127
    _set_token(a, 0, 400, 1, only, 0.01 * 2.0 ** octaves)
    a.call().launch(_stream())
    _check_elements(a, octaves, 8)


@pytest.mark.parametrize("seed", [0, 36, 136, 157, 161, 165])
def test_values_whose_scales_differ_by_sixty_orders_of_magnitude_between_tokens(dev, ws, seed):
    """Most elements are made up of few tokens; with the later seeds some of tokens further from the largest than exponentials reach."""
    torch.manual_seed(seed)
    for d, kv_heads in ((64, 2), (128, 2), (96, 1), (192, 1)):
        a = _Attention(dev, ws, rows=3, heads=4, kv_heads=kv_heads, d=d, block=16, lengths=[1, 40, 333], seed=13 + seed)
        s = a.p.scales[1]
        s.copy_(torch.exp(torch.rand_like(s) * 138 - 69))
        codes = a.p.codes[1]
        codes[torch.rand(codes.shape, device="cuda") < 0.7] = 0
        a.call().launch(_stream())
        _check_elements(a, 200, 4)


@pytest.mark.parametrize("d", [64, 128])
def test_many_equal_tokens_far_below_one(dev, ws, d):
    """Units that stay within one CTA, sixteen thousand tokens for a warp, all with the same small weight: whole numbers on the
    scale of the largest would round every one of them the same way."""
    rows, kv_heads, n, block = 320, 2, 64000, 16
    a = _Attention(dev, ws, rows=rows, heads=2 * kv_heads, kv_heads=kv_heads, d=d, block=block, lengths=[16] * rows, blocks=rows + 2, own_slots=True, unwritten=False, seed=4)
    rng = np.random.default_rng(5)
    table = np.concatenate(([0], rng.integers(1, rows, n // block - 1))).astype(np.int32)
    a.table = np.tile(table, (rows + 1, 1))
    a.positions = np.full(rows, n - 1, np.int32)
    _even_pages(a, 0.0)
    a.q[:] = a.q[0]
    gap = math.log(2.0 ** 27 / 0.4)
    a.p.codes[0, 0, :, 3] = 100
    a.p.scales[0, 0, :, 3] = gap / (100 * d * 0.5 * a.scale)
    a.p.codes[1, 0, :, 3] = torch.where(torch.arange(d, device="cuda") % 2 == 0, 100, 0).to(torch.int8)
    dq, dtable, dpos = (torch.from_numpy(x).cuda() for x in (a.q, a.table, a.positions))
    a.dq.copy_(dq)
    a.call(blockTable=dtable.data_ptr(), blocksPerSlot=n // block, positions=dpos.data_ptr()).launch(_stream())
    _check_elements(a, 0, n // 128, rows=[0, 100, rows - 1])


@pytest.mark.parametrize("rows,heads,kv_heads,d,n", [(1, 8, 2, 64, 1), (1, 8, 2, 64, 2), (4, 8, 8, 128, 20), (1, 8, 2, 64, 57), (2, 6, 2, 96, 100), (2, 16, 2, 128, 300), (1, 4, 1, 192, 300),
                                                     (1, 4, 1, 256, 700)])
def test_ordinary_rows_are_as_near_as_their_scores(dev, ws, rows, heads, kv_heads, d, n):
    """The norm of a head's error, without a term for long sums: each weight is off by the roundings of its score (three, and those of two differences
    that are no larger than the scores' own range), two exponentials (2^-22) and a few of 2^-24, as they come at random: a root of the sum of
    squares with uniform errors (1 / sqrt 3 of the largest), and three times that for the worst of these heads."""
    a = _Attention(dev, ws, rows=rows, heads=heads, kv_heads=kv_heads, d=d, block=16, lengths=[n] * rows, own_slots=True, unwritten=False, seed=n + d, spread=1.5)
    a.call().launch(_stream())
    torch.cuda.synchronize()
    got = a.out.cpu().numpy().astype(np.float64)
    for r in range(rows):
        for h in range(heads):
            s, want, _, _ = _terms(a, r, h)
            octaves = np.abs(s).max() / math.log(2)
            each = math.sqrt((3 * math.log(2) ** 2 * octaves ** 2 + 2 * (math.log(2) * 2 * octaves) ** 2 + 2 * 4 ** 2 + 4) / 3) * 2.0 ** -24
            assert np.linalg.norm(got[r, h * d:(h + 1) * d] - want) <= 3 * each * np.linalg.norm(want)
            assert abs(float(a.lse[r, h]) - (s.max() + math.log(np.exp(s - s.max()).sum()))) <= 3 * each + 2.0 ** -23 * np.abs(s).max()
