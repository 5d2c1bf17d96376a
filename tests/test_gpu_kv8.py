"""The 8-bit paged cache on the GPU against the plain statements of kv8_ref in 64 bits, through the public entry points."""
import math

import numpy as np
import pytest
import torch

import jitllm_b200 as jl
from jitllm_b200 import GGMLType
from tests import kv8_ref as ref

pytestmark = pytest.mark.gpu


def _up(x, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(x))
    return (t if dtype is None else t.to(dtype)).cuda()


def _stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.fixture(scope="module")
def ws(dev):
    w = jl.Kv8Workspace(dev)
    yield w
    w.close()


# ------------------------------------------------------------------------------------------------ map

class _Map:
    """Buffers of a map on the GPU and the plain statement's answer for them."""

    def __init__(self, ws, held, added, per, block, free, cursor, capacity, table=None, inplace=False, optional=True, seed=0):
        n = len(held)
        rng = np.random.default_rng(seed)
        if table is None:
            table = np.full((n, per), -1, np.int32)
            ids = 100000 + rng.permutation(n * per).astype(np.int32)
            for r in range(n):
                k = min(per, max(0, -(-int(held[r]) // block)))
                table[r, :k] = ids[r * per:r * per + k]
        self.want_table, self.n, self.inplace, self.optional = table.copy(), n, inplace, optional
        self.want_slots, self.want_pos = np.full(capacity, -7, np.int32), np.full(capacity, -7, np.int32)
        self.want_map = np.full(capacity, -7, np.int64)
        self.table, self.slots, self.pos, self.map = _up(table), _up(self.want_slots), _up(self.want_pos), _up(self.want_map)
        self.held, self.added = _up(np.asarray(held, np.int32)), _up(np.asarray(added, np.int32))
        self.free = _up(np.asarray(free, np.int32)) if len(free) else torch.zeros(1, dtype=torch.int32, device="cuda")
        self.cursor = torch.tensor([cursor], dtype=torch.int32, device="cuda")
        self.lengths = self.held if inplace else torch.zeros(n, dtype=torch.int32, device="cuda")
        self.cursor_out = self.cursor if inplace else torch.zeros(1, dtype=torch.int32, device="cuda")
        self.offsets = torch.full((n + 2,), -7, dtype=torch.int32, device="cuda")
        self.result = torch.full((5,), -7, dtype=torch.int32, device="cuda")
        self.lengths_want, self.offsets_want, self.cursor_want, self.result_want = ref.map_ref(
            held, added, self.want_table, np.asarray(free, np.int32), cursor, block, capacity, self.want_slots, self.want_pos, self.want_map)
        o = dict(offsets=self.offsets.data_ptr(), tokenSlots=self.slots.data_ptr(), positions=self.pos.data_ptr()) if optional else {}
        self.call = jl.Kv8Map(ws, held=self.held.data_ptr(), added=self.added.data_ptr(), sequences=n, blockTable=self.table.data_ptr(), blocksPerSlot=per,
                              blockSizeTokens=block, freeBlocks=self.free.data_ptr(), freeCount=len(free), cursor=self.cursor.data_ptr(),
                              cursorOut=self.cursor_out.data_ptr(), lengths=self.lengths.data_ptr(), slotMap=self.map.data_ptr(), capacity=capacity,
                              result=self.result.data_ptr(), **o)

    def check(self):
        torch.cuda.synchronize()
        assert np.array_equal(self.result.cpu().numpy(), np.append(self.result_want, -7))
        assert int(self.cursor_out) == self.cursor_want
        assert np.array_equal(self.lengths.cpu().numpy(), self.lengths_want)
        assert np.array_equal(self.table.cpu().numpy(), self.want_table)
        assert np.array_equal(self.map.cpu().numpy(), self.want_map)
        if self.optional:
            assert np.array_equal(self.offsets.cpu().numpy(), np.append(self.offsets_want, -7))
            assert np.array_equal(self.slots.cpu().numpy(), self.want_slots)
            assert np.array_equal(self.pos.cpu().numpy(), self.want_pos)


@pytest.mark.parametrize("n,block,most_added,short,seed", [
    (1, 16, 1, False, 0), (1, 1, 5, False, 1), (2, 16, 40, False, 2), (31, 16, 3, True, 3), (33, 7, 50, False, 4), (257, 16, 1, False, 5),
    (1000, 32, 90, True, 6), (1025, 16, 2, False, 7), (3413, 16, 3, False, 12), (3500, 16, 1, True, 13), (4096, 32, 5, False, 14), (4097, 16, 1, False, 15),
    (8192, 16, 9, False, 8), (8192, 64, 40, True, 9), (5, 65536, 100000, False, 10), (3, 16, 300000, False, 11)])
def test_map_of_random_batches(ws, n, block, most_added, short, seed):
    rng = np.random.default_rng(seed)
    held = rng.integers(0, 4 * block, n)
    added = rng.integers(0, most_added + 1, n)
    per = int(np.max(-(-(held + added) // block))) + 1
    need = int(np.sum(-(-(held + added) // block) - -(-held // block)))
    free = rng.permutation(need + 9)[:need + 3 if not short else max(1, need // 2)]
    m = _Map(ws, held, added, per, block, free, 3 if not short else 0, int(added.sum()) + 5, inplace=bool(seed % 2), seed=seed)
    m.call.launch(_stream())
    m.check()


def test_map_refuses_sequence_by_sequence(ws):
    """Negative lengths, no room in the row, tokens beyond the capacity, no blocks left: the others are served as if alone."""
    held = [5, -1, 30, 0, 16, 2**31 - 1, 0, 47, 9, 3]
    added = [3, 4, 19, -2, 1, 2**31 - 1, 0, 1, 200, 1]
    for capacity in (0, 6, 27, 60, 400):
        for free in (0, 1, 2, 5):
            m = _Map(ws, held, added, 3, 16, np.arange(free) + 70, 0, capacity)
            m.call.launch(_stream())
            m.check()


@pytest.mark.parametrize("cursor", [-1, 0, 3, 4, 5, 2**31 - 1])
def test_map_cursor_beyond_the_free_blocks_leaves_none(ws, cursor):
    m = _Map(ws, [0, 16, 3], [1, 1, 1], 4, 16, [8, 6, 4, 2], cursor, 9)
    m.call.launch(_stream())
    m.check()


def test_map_of_a_table_with_holes_and_without_optional_outputs(ws):
    table = np.array([[4, -1, 5, -1], [-1, -1, -1, -1]], np.int32)
    m = _Map(ws, [20, 6], [9, 3], 4, 16, [11, 12], 0, 20, table=table, optional=False)
    m.call.launch(_stream())
    m.check()


def test_map_step_by_step_in_place_in_a_graph(ws):
    """held and cursor are moved on by each replay: twenty decode steps of one captured call."""
    rng = np.random.default_rng(5)
    n, block, per = 37, 8, 12
    held = rng.integers(1, 40, n)
    free = rng.permutation(n * per)
    m = _Map(ws, held, np.ones(n, int), per, block, free, 0, n, inplace=True)
    table, cursor = m.table.cpu().numpy(), 0
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        m.call.launch(torch.cuda.current_stream().cuda_stream)
    for _ in range(20):
        slots, pos, place = np.empty(n, np.int32), np.empty(n, np.int32), np.empty(n, np.int64)
        held, _, cursor, _ = ref.map_ref(held, np.ones(n, int), table, free, cursor, block, n, slots, pos, place)
        g.replay()
        torch.cuda.synchronize()
        assert np.array_equal(m.map.cpu().numpy(), place) and np.array_equal(m.held.cpu().numpy(), held)
    assert np.array_equal(m.table.cpu().numpy(), table) and int(m.cursor) == cursor


# ------------------------------------------------------------------------------------------------ append

class _Pages:
    """Pages in memory with gaps between blocks, filled with random codes."""

    def __init__(self, dev, blocks, block, heads, d, seed=0, gap=0):
        rng = np.random.default_rng(seed)
        self.shape = (blocks, heads, block, d)
        stride, scale_stride = heads * block * d + 16 * gap, heads * block + gap
        self.raw = torch.from_numpy(rng.integers(-128, 128, (2, blocks * stride + 16)).astype(np.int8)).cuda()
        self.raw_scales = torch.from_numpy(rng.uniform(0.005, 0.03, (2, blocks * scale_stride + 16)).astype(np.float32)).cuda()
        view = lambda raw, shape, at: raw.as_strided(shape, (raw.stride(0), at, shape[3] * shape[4] if len(shape) == 5 else shape[3],  # noqa: E731
                                                             *((shape[4], 1) if len(shape) == 5 else (1,))))
        self.codes = view(self.raw, (2, blocks, heads, block, d), stride)
        self.scales = view(self.raw_scales, (2, blocks, heads, block), scale_stride)
        self.pages = jl.Kv8Pages(dev, self.codes[0].data_ptr(), self.codes[1].data_ptr(), self.scales[0].data_ptr(), self.scales[1].data_ptr(), blocks=blocks,
                                 blockSizeTokens=block, kvHeads=heads, headSize=d, blockStride=stride, scaleStride=scale_stride)

    def host(self):
        return self.codes.cpu().numpy().copy(), self.scales.cpu().numpy().astype(np.float64)


def _check_append(p, codes, scales):
    """Codes are those of the 64-bit values; a scale is the largest element (a rotation's roundings: 3 of 2^-24) over 127 in
    binary32 (2^-24): 2^-22."""
    torch.cuda.synchronize()
    got_codes, got_scales = p.host()
    assert np.array_equal(np.isnan(got_scales), np.isnan(scales))
    assert (np.abs(got_scales - scales)[~np.isnan(scales)] <= 2.0 ** -22 * scales[~np.isnan(scales)]).all()
    assert np.array_equal(got_codes, codes)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("rope", [False, True])
@pytest.mark.parametrize("d,heads,block,tokens,gap", [(64, 2, 16, 1, 0), (64, 1, 1, 7, 0), (96, 3, 5, 33, 1), (128, 8, 16, 300, 0), (192, 2, 32, 65, 3),
                                                      (256, 1, 16, 40, 0), (128, 5, 64, 1030, 0)])
def test_append(dev, f16, rope, d, heads, block, tokens, gap):
    rng = np.random.default_rng(d + tokens)
    p = _Pages(dev, -(-tokens // block) + 3, block, heads, d, seed=tokens, gap=gap)
    codes, scales = p.host()
    dtype = np.float16 if f16 else np.float32
    joint = (rng.standard_normal((tokens, 2 * heads * d + 16)) * np.exp(2 * rng.standard_normal((tokens, 1)))).astype(dtype)
    k, v = joint[:, :heads * d], joint[:, heads * d:2 * heads * d]
    slot_map = rng.permutation(p.shape[0] * block)[:tokens].astype(np.int64)
    positions = rng.integers(0, 5000, tokens).astype(np.int32)
    cos, sin = ref.rope_tables(5000, d)
    ref.append_ref(codes, scales, k, v, slot_map, tokens, positions, cos if rope else None, sin)
    x, m, pos, c, s = _up(joint), _up(slot_map), _up(positions), _up(cos), _up(sin)
    jl.Kv8Append(p.pages, x.data_ptr(), x[:, heads * d:].data_ptr(), GGMLType.F16 if f16 else GGMLType.F32, tokens=tokens, slotMap=m.data_ptr(),
                 keyStride=x.stride(0), valueStride=x.stride(0), positions=pos.data_ptr(),
                 **(dict(ropeCos=c.data_ptr(), ropeSin=s.data_ptr(), ropeRows=5000) if rope else {})).launch(_stream())
    before = p.raw.clone()
    _check_append(p, codes, scales)
    assert torch.equal(before, p.raw)
    if gap:  # nothing is written between blocks
        untouched = np.random.default_rng(tokens).integers(-128, 128, tuple(p.raw.shape)).astype(np.int8)
        stride = p.codes.stride(1)
        raw = p.raw.cpu().numpy()[:, :p.shape[0] * stride].reshape(2, p.shape[0], stride)
        assert np.array_equal(raw[:, :, -16 * gap:], untouched[:, :p.shape[0] * stride].reshape(2, p.shape[0], stride)[:, :, -16 * gap:])


def test_append_passes_over_what_has_no_place(dev):
    """Places outside the pages, rows behind the token count, positions outside the tables, rows of zeros, infinities, NaN."""
    d, heads, block, tokens, rows = 128, 4, 16, 24, 30
    rng = np.random.default_rng(4)
    p = _Pages(dev, 4, block, heads, d, seed=9)
    codes, scales = p.host()
    k, v = (rng.standard_normal((rows, heads, d)).astype(np.float32) for _ in range(2))
    k[0], v[1, 2], k[2, 1] = 0, 0, 1e-38
    k[3, 0, 5], v[3, 1, 127], k[4, 2, 0], v[4, 3, 64] = np.inf, -np.inf, np.nan, np.nan
    v[5, 0], v[6, 0, 7] = 3e38, 3.4e38
    v[7, 1], v[7, 2] = 2.0 ** -100, np.float32(2.0 ** -100) * np.float32(0.9999999)
    slot_map = rng.permutation(4 * block)[:rows].astype(np.int64)
    slot_map[[10, 11, 12, 13]] = -1, 4 * block, -2 ** 62, 2 ** 40
    positions = np.arange(rows).astype(np.int32)
    positions[[14, 15, 16]] = -1, 40, 2 ** 31 - 1
    cos, sin = ref.rope_tables(40, d)
    ref.append_ref(codes, scales, k, v, slot_map, tokens, positions, cos, sin)
    x, y, m, pos, c, s, n = _up(k), _up(v), _up(slot_map), _up(positions), _up(cos), _up(sin), torch.tensor([tokens], dtype=torch.int32, device="cuda")
    call = jl.Kv8Append(p.pages, x.data_ptr(), y.data_ptr(), GGMLType.F32, tokens=rows, slotMap=m.data_ptr(), positions=pos.data_ptr(), ropeCos=c.data_ptr(),
                        ropeSin=s.data_ptr(), ropeRows=40, tokenCount=n.data_ptr())
    call.launch(_stream())
    _check_append(p, codes, scales)
    for count in (0, -5):
        n.fill_(count)
        before = p.raw.clone()
        call.launch(_stream())
        torch.cuda.synchronize()
        assert torch.equal(before, p.raw)
    n.fill_(10 ** 6)  # more than the rows there are: all of them
    call.launch(_stream())
    ref.append_ref(codes, scales, k, v, slot_map, rows, positions, cos, sin)
    _check_append(p, codes, scales)


def test_append_codes_next_to_the_border_of_two(dev):
    """Elements within a few roundings of half a code, ties among them, plain and rotated."""
    d, heads, block, tokens = 128, 2, 16, 512
    rng = np.random.default_rng(12)
    p = _Pages(dev, tokens // block, block, heads, d)
    codes, scales = p.host()
    most = np.exp(rng.standard_normal((tokens, heads, 1)))
    most[::4] = 127.0 * 2.0 ** rng.integers(-8, 9, (len(most[::4]), heads, 1))  # ties are exact
    x = ((rng.integers(-127, 127, (tokens, heads, d)) + 0.5) * most / 127).astype(np.float32)
    x = np.nextafter(x, np.where(rng.random(x.shape) < 0.3, np.inf, np.where(rng.random(x.shape) < 0.4, -np.inf, x)).astype(np.float32))
    x[:, :, 5:6] = most
    slot_map = np.arange(tokens, dtype=np.int64)
    positions = rng.integers(0, 999, tokens).astype(np.int32)
    cos, sin = ref.rope_tables(999, d)
    back = ref.rotate(x.astype(np.float64), cos[positions].astype(np.float64)[:, None], -sin[positions].astype(np.float64)[:, None]).astype(np.float32)
    ref.append_ref(codes, scales, back, x, slot_map, tokens, positions, cos, sin)
    k, v, m, pos, c, s = _up(back), _up(x), _up(slot_map), _up(positions), _up(cos), _up(sin)
    jl.Kv8Append(p.pages, k.data_ptr(), v.data_ptr(), GGMLType.F32, tokens=tokens, slotMap=m.data_ptr(), positions=pos.data_ptr(), ropeCos=c.data_ptr(),
                 ropeSin=s.data_ptr(), ropeRows=999).launch(_stream())
    _check_append(p, codes, scales)


def test_append_at_places_beyond_32_bits(dev):
    """The last block of pages of more than 2^32 bytes."""
    d, heads, block, blocks = 128, 8, 64, 66000
    raw = torch.zeros((2, blocks, heads, block, d), dtype=torch.int8, device="cuda")
    scales = torch.zeros((2, blocks, heads, block), device="cuda")
    pages = jl.Kv8Pages(dev, raw[0].data_ptr(), raw[1].data_ptr(), scales[0].data_ptr(), scales[1].data_ptr(), blocks=blocks, blockSizeTokens=block, kvHeads=heads,
                        headSize=d)
    rng = np.random.default_rng(1)
    k, v = (rng.standard_normal((2, heads, d)).astype(np.float32) for _ in range(2))
    place = np.array([blocks * block - 1, (blocks - 1) * block], np.int64)
    x, y, m = _up(k), _up(v), _up(place)
    jl.Kv8Append(pages, x.data_ptr(), y.data_ptr(), GGMLType.F32, tokens=2, slotMap=m.data_ptr()).launch(_stream())
    for which, want in ((0, k), (1, v)):
        codes, sc = ref.quantise(want)
        got = raw[which, -1][:, [63, 0]].cpu().numpy().transpose(1, 0, 2)
        assert np.array_equal(got, codes)
        assert np.allclose(scales[which, -1][:, [63, 0]].cpu().numpy().T, sc, rtol=2 ** -23, atol=0)
    assert int(torch.count_nonzero(scales)) == 4 * heads


# ------------------------------------------------------------------------------------------------ attention

class _Attention:
    def __init__(self, dev, ws, *, rows, heads, kv_heads, d, block, lengths, window=0, f16=False, rope=False, blocks=None, gap=0, pad=0, lse=True, seed=0,
                 scale=None, own_slots=False, holes=0.0, spread=1.0, unwritten=True):
        rng = np.random.default_rng(seed)
        self.rng = rng
        lengths = np.asarray(lengths)
        per = max(1, int(np.max(-(-np.maximum(lengths, 0) // block)))) + 1
        have = -(-np.maximum(lengths, 0) // block)
        blocks = blocks or int(have.sum()) + 2
        self.p = _Pages(dev, blocks, block, kv_heads, d, seed=seed, gap=gap)
        ids = rng.permutation(blocks)[:int(have.sum())]
        self.table = np.full((rows + 1, per), -1, np.int32)
        order = np.arange(rows) if own_slots else rng.permutation(rows + 1)[:rows]
        at = 0
        scales = self.p.scales.cpu().numpy()
        for r in range(rows):
            mine = ids[at:at + have[r]]
            at += have[r]
            self.table[order[r], :have[r]] = mine
            if have[r] and unwritten and lengths[r] % block:  # what no token has been written to holds anything
                scales[:, mine[-1], :, lengths[r] % block:] = np.nan
        if holes:
            gone = rng.random(self.table.shape) < holes
            self.table[gone] = rng.choice([-1, blocks, 2 ** 31 - 1, -2 ** 31], int(gone.sum()))
        self.p.scales.copy_(torch.from_numpy(scales).cuda())
        self.kv_slots = None if own_slots else order.astype(np.int32)
        self.positions = (lengths - 1).astype(np.int32)
        dtype = np.float16 if f16 else np.float32
        self.q = np.zeros((rows, heads * d + pad), dtype)
        self.q[:, :heads * d] = rng.standard_normal((rows, heads * d)) * spread
        self.rows, self.heads, self.d, self.f16, self.window, self.block = rows, heads, d, f16, window, block
        self.scale = d ** -0.5 if scale is None else scale
        limit = int(max(1, lengths.max()))
        self.cos, self.sin = ref.rope_tables(limit, d) if rope else (None, None)
        self.dq, self.dtable, self.dpos = _up(self.q), _up(self.table), _up(self.positions)
        self.dslots = None if self.kv_slots is None else _up(self.kv_slots)
        self.out = torch.full((rows, heads * d + pad), 77.0, dtype=self.dq.dtype, device="cuda")
        self.lse = torch.full((rows, heads), 77.0, device="cuda") if lse else None
        self.count = None
        kw = {}
        if rope:
            self.dcos, self.dsin = _up(self.cos), _up(self.sin)
            kw = dict(ropeCos=self.dcos.data_ptr(), ropeSin=self.dsin.data_ptr(), ropeRows=limit)
        self.kw = dict(rows=rows, heads=heads, blockTable=self.dtable.data_ptr(), slots=rows + 1, blocksPerSlot=per, positions=self.dpos.data_ptr(),
                       kvSlots=0 if self.dslots is None else self.dslots.data_ptr(), lse=self.lse.data_ptr() if lse else 0, queryStride=self.dq.stride(0),
                       outStride=self.out.stride(0), window=window, scale=scale, **kw)
        self.ws = ws

    def call(self, **changes):
        return jl.Kv8Attention(self.p.pages, self.ws, self.dq.data_ptr(), self.out.data_ptr(), GGMLType.F16 if self.f16 else GGMLType.F32, **{**self.kw, **changes})

    def want(self, count=None):
        codes, scales = self.p.host()
        q = self.q[:, :self.heads * self.d].reshape(self.rows, self.heads, self.d)
        return ref.attention_ref(codes, scales, q, self.table, self.kv_slots, self.positions, self.scale, self.window, self.cos, self.sin, count)

    def check(self, want=None, count=None):
        torch.cuda.synchronize()
        out, lse, most = want or self.want(count)
        n = self.rows if count is None else count
        got = self.out.float().cpu().numpy().astype(np.float64)
        assert (got[:, self.heads * self.d:] == 77).all() and (got[n:] == 77).all()
        got = got[:n, :self.heads * self.d].reshape(n, self.heads, self.d)
        out, lse = out[:n], lse[:n]
        assert np.array_equal(np.isnan(got), np.isnan(out))
        for r in range(n):
            assert not got[r][out[r] == 0].any() or out[r].any()
            fine = ~np.isnan(out[r])
            far = np.linalg.norm((got[r] - out[r])[fine])
            # scores by score_tolerance; the weights' rounding and sums as many again; binary16 rounds each output by 2^-11 of it (or 2^-25)
            tol = 2 * ref.score_tolerance(self.d, most[r]) * np.linalg.norm(out[r][fine])
            if self.f16:
                tol += 2.0 ** -11 * np.linalg.norm(out[r][fine]) + 2.0 ** -25 * math.sqrt(fine.sum())
            assert far <= tol, (r, far, tol)
            if self.lse is not None:
                x = self.lse[r].cpu().numpy().astype(np.float64)
                assert np.array_equal(np.isnan(x), np.isnan(lse[r])) and np.array_equal(np.isinf(x), np.isinf(lse[r]))
                ok = np.isfinite(lse[r])
                assert (np.abs(x[ok] - lse[r][ok]) <= ref.score_tolerance(self.d, most[r]) + 2.0 ** -23 * np.abs(lse[r][ok])).all()


LENGTHS = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 100, 127, 128, 129, 255, 257, 300]


@pytest.mark.parametrize("d,heads,kv_heads", [(64, 8, 2), (64, 3, 3), (96, 6, 2), (128, 32, 8), (128, 7, 1), (128, 16, 1), (128, 40, 2), (192, 10, 2), (256, 8, 1),
                                              (256, 4, 4), (128, 9, 1), (64, 64, 4)])
@pytest.mark.parametrize("f16,rope", [(False, False), (False, True), (True, True)])
def test_attention_of_ragged_rows(dev, ws, d, heads, kv_heads, f16, rope):
    a = _Attention(dev, ws, rows=len(LENGTHS), heads=heads, kv_heads=kv_heads, d=d, block=16, lengths=LENGTHS, f16=f16, rope=rope, seed=d + heads, pad=16, gap=1)
    a.call().launch(_stream())
    a.check()


@pytest.mark.parametrize("block", [1, 3, 5, 16, 24, 32, 64, 100, 1000])
@pytest.mark.parametrize("window", [0, 1, 17, 64, 150])
def test_attention_of_pages_that_end_anywhere_and_windows(dev, ws, block, window):
    a = _Attention(dev, ws, rows=9, heads=8, kv_heads=2, d=64, block=block, lengths=[0, 1, 40, 64, 65, 149, 150, 151, 311], window=window, rope=True, seed=block)
    a.call().launch(_stream())
    a.check()


@pytest.mark.parametrize("rows,heads,kv_heads,d,lengths", [
    (1, 8, 2, 64, [57]), (1, 32, 8, 128, [3901]), (1, 8, 1, 128, [20001]), (2, 1, 1, 64, [50000, 3]), (4, 32, 8, 128, [1, 9000, 20, 3000]),
    (1, 1, 1, 256, [7777]), (70, 16, 8, 128, [700] * 70), (3, 16, 1, 64, [12345, 6789, 4097]), (300, 4, 1, 64, list(range(300)))])
def test_attention_of_long_and_wide_batches(dev, ws, rows, heads, kv_heads, d, lengths):
    a = _Attention(dev, ws, rows=rows, heads=heads, kv_heads=kv_heads, d=d, block=16, lengths=lengths, rope=True, seed=rows, spread=1.5)
    a.call().launch(_stream())
    want = a.want()
    a.check(want)
    first, lse = a.out.clone(), a.lse.clone()
    for _ in range(3):  # no result hangs on the order in which blocks of a grid arrive
        a.out.fill_(77.0)
        a.call().launch(_stream())
        torch.cuda.synchronize()
        assert torch.equal(first, a.out) and torch.equal(lse, a.lse)


def test_attention_with_holes_and_bad_entries_of_the_table(dev, ws):
    """Entries that are no block of the pages are passed over; sequences outside the table and negative positions see nothing."""
    a = _Attention(dev, ws, rows=12, heads=8, kv_heads=2, d=128, block=16, lengths=[900, 5, 16, 17, 100, 200, 300, 0, 64, 90, 33, 48], holes=0.4, seed=5, rope=True)
    a.kv_slots[[4, 5, 9]] = -1, 13, 2 ** 31 - 1
    a.positions[[8, 10]] = -2 ** 31, -7
    a.dslots.copy_(_up(a.kv_slots))
    a.dpos.copy_(_up(a.positions))
    a.call().launch(_stream())
    a.check()
    assert (a.lse[4] == -math.inf).all() and (a.lse[5] == -math.inf).all() and not a.out[8, :1024].any()
    a.dtable.fill_(-1)
    a.table[:] = -1
    a.call().launch(_stream())
    a.check()
    assert not a.out[:, :1024].any() and (a.lse == -math.inf).all()


def test_attention_at_positions_beyond_the_table_and_the_rotation(dev, ws):
    a = _Attention(dev, ws, rows=4, heads=4, kv_heads=2, d=64, block=16, lengths=[20, 40, 33, 48], rope=True, own_slots=True, seed=3, unwritten=False)
    a.positions[:] = 19, 2 ** 31 - 1, 32, 400   # rows hold 4 blocks of 16
    a.dpos.copy_(_up(a.positions))
    a.call().launch(_stream())
    a.check()                                   # rows 1 and 3: rotated beyond the tables, NaN
    assert torch.isnan(a.out[1]).all() and torch.isnan(a.out[3]).all()
    a.cos = a.sin = None
    a.window = 2 ** 31 - 1
    a.call(ropeCos=0, ropeSin=0, window=a.window).launch(_stream())
    a.check()
    assert torch.isfinite(a.out).all()
    a.window = 100                              # the window of row 1 lies behind the table
    a.call(ropeCos=0, ropeSin=0, window=a.window).launch(_stream())
    a.check()
    assert (a.lse[1] == -math.inf).all()


def test_attention_leaves_rows_behind_the_count(dev, ws):
    a = _Attention(dev, ws, rows=8, heads=8, kv_heads=4, d=64, block=16, lengths=[100, 2000, 30, 4, 500, 60, 70, 80], seed=6)
    n = torch.tensor([3], dtype=torch.int32, device="cuda")
    a.call(tokenCount=n.data_ptr()).launch(_stream())
    a.check(count=3)
    for count in (0, -4):
        n.fill_(count)
        a.out.fill_(77.0)
        a.call(tokenCount=n.data_ptr()).launch(_stream())
        torch.cuda.synchronize()
        assert (a.out == 77).all()
    n.fill_(1 << 30)
    a.call(tokenCount=n.data_ptr()).launch(_stream())
    a.check()
    a.call(rows=0).launch(_stream())


def test_attention_of_shared_blocks_and_rows_of_one_sequence(dev, ws):
    """Several tokens of one sequence, each seeing what is before it, and sequences that share their first blocks."""
    a = _Attention(dev, ws, rows=6, heads=4, kv_heads=2, d=128, block=16, lengths=[70, 71, 72, 73, 300, 300], seed=8, unwritten=False)
    a.kv_slots[:4] = a.kv_slots[3]
    a.table[a.kv_slots[5], :7] = a.table[a.kv_slots[4], :7]
    a.dslots.copy_(_up(a.kv_slots))
    a.dtable.copy_(_up(a.table))
    a.call().launch(_stream())
    a.check()


@pytest.mark.parametrize("spread,scale", [(1e-4, None), (40.0, None), (1e4, 1e-5), (1.0, 0.0), (1.0, -0.3), (1e-30, 1e29), (3e30, 1e-31), (2.0 ** -130, 1e37)])
def test_attention_of_small_and_large_queries_and_scales(dev, ws, spread, scale):
    a = _Attention(dev, ws, rows=3, heads=8, kv_heads=2, d=128, block=16, lengths=[1, 77, 1500], seed=11, spread=spread, scale=scale)
    a.call().launch(_stream())
    a.check()


def test_attention_of_queries_whose_elements_differ_in_size(dev, ws):
    """Heads of one row a million times larger than others, and elements of one head."""
    a = _Attention(dev, ws, rows=2, heads=8, kv_heads=1, d=128, block=16, lengths=[500, 90], seed=12)
    a.q[:, :1024] *= np.repeat(10.0 ** np.arange(-7, 1), 128).astype(np.float32)
    a.q[1, :1024] *= np.exp(np.random.default_rng(2).standard_normal(1024) * 4).astype(np.float32)
    a.dq.copy_(_up(a.q))
    a.call().launch(_stream())
    a.check()


def test_attention_of_values_of_very_different_size(dev, ws):
    """Scales of values over sixty orders of magnitude between tokens: every weight times its scale keeps its 24 bits."""
    for d in (64, 128):
        a = _Attention(dev, ws, rows=4, heads=4, kv_heads=2, d=d, block=16, lengths=[1, 40, 333, 2000], seed=13)
        s = a.p.scales[1]
        s.copy_(torch.exp(torch.rand_like(s) * 138 - 69))
        a.call().launch(_stream())
        a.check()
        s.fill_(1e-30)
        a.call().launch(_stream())
        a.check()
        s.fill_(2e36)
        a.call().launch(_stream())
        a.check()


def test_attention_nan_reaches_the_heads_that_read_it_and_no_others(dev, ws):
    a = _Attention(dev, ws, rows=3, heads=8, kv_heads=2, d=64, block=16, lengths=[50, 1000, 200], seed=14)
    a.p.scales[0, a.table[a.kv_slots[0], 1], 1, 3] = math.nan     # a key of row 0, KV head 1
    a.p.scales[1, a.table[a.kv_slots[1], 30], 0, 2] = math.nan    # a value of row 1, KV head 0
    a.q[2, 5 * 64 + 9] = np.nan                                   # query head 5 of row 2
    a.dq.copy_(_up(a.q))
    a.call().launch(_stream())
    a.check()
    assert torch.isnan(a.out[0, 4 * 64:8 * 64]).all() and torch.isfinite(a.out[0, :4 * 64]).all()
    assert torch.isnan(a.out[1, :4 * 64]).all() and torch.isfinite(a.out[1, 4 * 64:]).all()
    assert torch.isnan(a.out[2, 5 * 64:6 * 64]).all() and torch.isfinite(a.out[2, :5 * 64]).all() and torch.isfinite(a.out[2, 6 * 64:]).all()


def test_attention_of_a_peaked_row_and_of_equal_scores(dev, ws):
    a = _Attention(dev, ws, rows=2, heads=4, kv_heads=1, d=64, block=16, lengths=[3000, 3000], seed=15, spread=60.0)
    a.q[1] = 0
    a.dq.copy_(_up(a.q))
    a.call().launch(_stream())
    a.check()


def test_attention_in_pages_beyond_32_bits(dev, ws):
    """Blocks at the end of pages of more than 2^32 bytes, and a table whose entries are all over them."""
    d, heads, block, blocks, n = 128, 8, 64, 66000, 3000
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    raw = torch.zeros((2, blocks, heads, block, d), dtype=torch.int8, device="cuda")
    scales = torch.zeros((2, blocks, heads, block), device="cuda")
    ids = torch.cat((torch.tensor([blocks - 1, 0, blocks - 2]), torch.randperm(blocks - 3)[:44] + 1)).cuda()
    raw[:, ids] = torch.randint(-127, 128, (2, 47, heads, block, d), device="cuda", generator=g, dtype=torch.int8)
    scales[:, ids] = torch.rand((2, 47, heads, block), device="cuda", generator=g) * 0.02 + 0.005
    pages = jl.Kv8Pages(dev, raw[0].data_ptr(), raw[1].data_ptr(), scales[0].data_ptr(), scales[1].data_ptr(), blocks=blocks, blockSizeTokens=block, kvHeads=heads,
                        headSize=d)
    q, table, pos = torch.randn((1, 16 * d), device="cuda", generator=g), ids.int().view(1, -1).contiguous(), torch.tensor([n - 1], dtype=torch.int32, device="cuda")
    out = torch.empty((1, 16, d), device="cuda")
    jl.Kv8Attention(pages, ws, q.data_ptr(), out.data_ptr(), GGMLType.F32, rows=1, heads=16, blockTable=table.data_ptr(), slots=1, blocksPerSlot=47,
                    positions=pos.data_ptr()).launch(_stream())
    want, _, most = ref.attention_ref(raw[:, ids].cpu().numpy(), scales[:, ids].cpu().numpy(), q.view(1, 16, d).cpu().numpy(), np.arange(47)[None], None, [n - 1],
                                      d ** -0.5)
    assert np.linalg.norm(out.cpu().numpy() - want) <= 2 * ref.score_tolerance(d, most[0]) * np.linalg.norm(want)


def test_attention_of_a_long_sequence_of_repeated_blocks(dev, ws):
    """More steps for a warp than its integer sums hold at once (2^16 tokens): the blocks of a row repeat, so that the output is that of
    one round of them, and its lse that and the logarithm of the rounds."""
    rows, heads, d, block, rounds = 64, 8, 64, 16, 5000
    p = _Pages(dev, 4, block, heads, d, seed=3)
    rng = np.random.default_rng(3)
    q = rng.standard_normal((rows, heads, d)).astype(np.float32)
    table = np.tile(np.arange(4, dtype=np.int32), rounds)[None].repeat(rows, 0)
    x, tab, pos = _up(q), _up(table), _up(np.full(rows, 4 * block * rounds - 1, np.int32))
    out, lse = torch.empty((rows, heads, d), device="cuda"), torch.empty((rows, heads), device="cuda")
    jl.Kv8Attention(p.pages, ws, x.data_ptr(), out.data_ptr(), GGMLType.F32, rows=rows, heads=heads, blockTable=tab.data_ptr(), slots=rows,
                    blocksPerSlot=4 * rounds, positions=pos.data_ptr(), lse=lse.data_ptr()).launch(_stream())
    codes, scales = p.host()
    want, want_lse, most = ref.attention_ref(codes, scales, q, table[:, :4], None, np.full(rows, 4 * block - 1), d ** -0.5)
    torch.cuda.synchronize()
    tol = 2 * ref.score_tolerance(d, most.max())
    assert np.linalg.norm(out.cpu().numpy() - want) <= tol * np.linalg.norm(want)
    # a warp's sum of weights has 2 000 steps of four tokens for a lane, each addition off by 2^-24 of it
    assert np.abs(lse.cpu().numpy() - want_lse - math.log(rounds)).max() <= tol + 2.0 ** -24 * 4 * 2200 + 2.0 ** -22 * 20


@pytest.mark.parametrize("gap", [3.0, 8.0, 12.0, 25.0])
def test_attention_with_a_token_far_above_the_others(dev, ws, gap):
    """One token's weight is e^gap times the others': these keep their part of the output, wherever the one stands."""
    for at in (0, 777, 2999):
        a = _Attention(dev, ws, rows=1, heads=8, kv_heads=2, d=128, block=16, lengths=[3000], seed=16, spread=0.3, own_slots=True, unwritten=False)
        codes = a.p.codes
        b, place = int(a.table[0, at // 16]), at % 16
        for h in range(2):
            codes[0, b, h, place] = 100
            a.p.scales[0, b, h, place] = gap / (100 * 0.3 * 128 ** 0.5) * 128 ** 0.5 / 128
        a.q[0, :1024] = np.abs(a.q[0, :1024]) + 0.3
        a.dq.copy_(_up(a.q))
        a.call().launch(_stream())
        a.check()


@pytest.mark.parametrize("rows", [33, 128, 129, 1000])
def test_attention_of_many_rows_some_of_them_long(dev, ws, rows):
    """Rows beyond those that a warp's lanes hold, in front of and behind long ones."""
    rng = np.random.default_rng(rows)
    lengths = rng.integers(0, 90, rows)
    lengths[[0, rows // 2, rows - 1]] = 3000, 5000, 2100
    a = _Attention(dev, ws, rows=rows, heads=4, kv_heads=2, d=64, block=16, lengths=lengths, seed=rows, rope=True)
    a.call().launch(_stream())
    a.check()


def test_attention_of_groups_of_more_heads_than_the_grid_has_places(dev, ws):
    a = _Attention(dev, ws, rows=2, heads=4096, kv_heads=1, d=128, block=16, lengths=[300, 40], seed=17)
    a.call().launch(_stream())
    a.check()


# ------------------------------------------------------------------------------------------------ calls

@pytest.mark.parametrize("heads,kv_heads,d,block,n", [(6, 6, 192, 48, 700), (12, 2, 96, 7, 5000)])
def test_the_first_call_of_a_kind_may_be_captured(dev, heads, kv_heads, d, block, n):
    """Nothing that a first call sets up is in a capture's way; two graphs with one workspace, replayed in turn."""
    w = jl.Kv8Workspace(dev)
    a = [_Attention(dev, w, rows=3, heads=heads, kv_heads=kv_heads, d=d, block=block, lengths=[n, 5, n // 2 + k], seed=k) for k in range(2)]
    graphs = []
    for x in a:
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            x.call().launch(torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    for _ in range(3):
        for x, g in zip(a, graphs):
            x.out.fill_(77.0)
            g.replay()
    for x in a:
        x.check()
    del g, graphs
    w.close()


def test_closed_workspaces_and_devices_refuse(dev):
    d = jl.Device(0)
    w = jl.Kv8Workspace(d)
    a = _Attention(d, w, rows=1, heads=4, kv_heads=2, d=64, block=16, lengths=[20])
    call = a.call()
    call.launch()
    d.synchronize()
    w.close()
    with pytest.raises(jl.IllegalStateError, match="closed"):
        call.launch()
    with jl.Kv8Workspace(d) as again:
        call.workspace = again
        call.launch()
        d.synchronize()
        d.close()
        with pytest.raises(jl.IllegalStateError, match="closed"):
            call.launch()
    a.check()


def test_refused_calls_raise_and_launch_nothing(dev, ws):
    a = _Attention(dev, ws, rows=1, heads=4, kv_heads=2, d=64, block=16, lengths=[20])
    before = dev.counters()["kernel_launches"]
    with pytest.raises(ValueError, match="heads"):
        a.call(heads=3).launch(_stream())
    with pytest.raises(ValueError, match="window"):
        a.call(window=-1).launch()
    with pytest.raises(ValueError, match="GGML type 8"):
        jl.Kv8Attention(a.p.pages, ws, a.dq.data_ptr(), a.out.data_ptr(), GGMLType.Q8_0, **a.kw).launch()
    with jl.Device(0) as other:
        foreign = jl.Kv8Workspace(other)
        call = a.call()
        call.workspace = foreign
        with pytest.raises(ValueError, match="workspace"):
            call.launch()
        foreign.close()
        with pytest.raises(jl.IllegalStateError):
            call.launch()
    assert dev.counters()["kernel_launches"] == before
    torch.cuda.synchronize()
    assert (a.out == 77).all()


def test_calls_on_the_contexts_stream_on_others_and_at_once(dev):
    """Two streams with a workspace each, many calls of different shapes in flight on both."""
    w = [jl.Kv8Workspace(dev) for _ in range(2)]
    a = [_Attention(dev, w[0], rows=5, heads=8, kv_heads=2, d=128, block=16, lengths=[5000, 1, 300, 40, 2500], seed=21),
         _Attention(dev, w[1], rows=40, heads=4, kv_heads=4, d=64, block=16, lengths=list(range(0, 2000, 50)), seed=22)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(30):
        for x, s in zip(a, streams):
            x.call().launch(s.cuda_stream)
    for x in a:
        x.check()
    for x in a:
        x.out.fill_(77.0)
    torch.cuda.synchronize()
    for x in a:
        x.call().launch()
    dev.synchronize()
    for x in a:
        x.check()
    for x in w:
        x.close()


def test_a_step_of_all_three_eager_and_in_a_graph(dev):
    """Prompts, then decode steps: map -> append -> attention on the device, with rows behind the last token, replayed as one graph;
    against the plain statements in the same order, whose pages are the quantised ones."""
    rng = np.random.default_rng(31)
    n, per, block, heads, kv_heads, d, capacity = 5, 20, 16, 8, 2, 128, 64
    blocks = 60
    w = jl.Kv8Workspace(dev)
    p = _Pages(dev, blocks, block, kv_heads, d, seed=1)
    codes, scales = p.host()
    cos, sin = ref.rope_tables(per * block, d)
    free = rng.permutation(blocks).astype(np.int32)
    table, held, cursor = np.full((n, per), -1, np.int32), np.zeros(n, np.int32), 0
    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32, device="cuda")  # noqa: E731
    g = dict(held=i32(n), added=i32(n), free=_up(free), cursor=i32(1), table=_up(table), offsets=i32(n + 1), slots=i32(capacity), pos=i32(capacity),
             map=torch.zeros(capacity, dtype=torch.int64, device="cuda"), result=i32(4), qkv=torch.zeros((capacity, (heads + 2 * kv_heads) * d), device="cuda"),
             out=torch.zeros((capacity, heads, d), device="cuda"), cos=_up(cos), sin=_up(sin))
    at = {k: t.data_ptr() for k, t in g.items()}
    rope = dict(ropeCos=at["cos"], ropeSin=at["sin"], ropeRows=per * block)
    calls = [jl.Kv8Map(w, held=at["held"], added=at["added"], sequences=n, blockTable=at["table"], blocksPerSlot=per, blockSizeTokens=block, freeBlocks=at["free"],
                       freeCount=blocks, cursor=at["cursor"], cursorOut=at["cursor"], lengths=at["held"], offsets=at["offsets"], tokenSlots=at["slots"],
                       positions=at["pos"], slotMap=at["map"], capacity=capacity, result=at["result"]),
             jl.Kv8Append(p.pages, at["qkv"] + 4 * heads * d, at["qkv"] + 4 * (heads + kv_heads) * d, GGMLType.F32, tokens=capacity, slotMap=at["map"],
                          keyStride=g["qkv"].stride(0), valueStride=g["qkv"].stride(0), positions=at["pos"], tokenCount=at["result"], **rope),
             jl.Kv8Attention(p.pages, w, at["qkv"], at["out"], GGMLType.F32, rows=capacity, heads=heads, blockTable=at["table"], slots=n, blocksPerSlot=per,
                             kvSlots=at["slots"], positions=at["pos"], queryStride=g["qkv"].stride(0), tokenCount=at["result"], **rope)]
    graph = None
    for step in range(12):
        added = rng.integers(1, 13, n) if step == 0 else rng.choice([0, 1, 1, 1, 5], n) if step < 10 else np.array([0, 0, 7, 1, 0])
        total = int(added.sum())
        qkv = rng.standard_normal((capacity, (heads + 2 * kv_heads) * d)).astype(np.float32)
        g["added"].copy_(torch.from_numpy(added.astype(np.int32)))
        g["qkv"].copy_(torch.from_numpy(qkv))
        g["out"].fill_(7)
        slots, pos, place = np.zeros(capacity, np.int32), np.zeros(capacity, np.int32), np.zeros(capacity, np.int64)
        held, _, cursor, result = ref.map_ref(held, added, table, free, cursor, block, capacity, slots, pos, place)
        k, v = qkv[:, heads * d:(heads + kv_heads) * d], qkv[:, (heads + kv_heads) * d:]
        ref.append_ref(codes, scales, k, v, place, total, pos, cos, sin)
        want, _, most = ref.attention_ref(codes, scales.astype(np.float32), qkv[:total, :heads * d].reshape(total, heads, d), table, slots, pos[:total], d ** -0.5,
                                          cos=cos, sin=sin)
        if step < 4:
            for c in calls:
                c.launch(_stream())
        else:
            if graph is None:
                graph = torch.cuda.CUDAGraph()
                torch.cuda.synchronize()
                with torch.cuda.graph(graph):
                    for c in calls:
                        c.launch(torch.cuda.current_stream().cuda_stream)
            graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(g["result"].cpu().numpy(), result) and np.array_equal(g["table"].cpu().numpy(), table)
        got = g["out"].cpu().numpy()
        assert (got[total:] == 7).all()
        # scales differ by 2^-22 between the two sides: scores and values by as much
        far, norm = np.linalg.norm(got[:total] - want), np.linalg.norm(want)
        assert far <= (2 * ref.score_tolerance(d, most.max()) + 2.0 ** -21 * (1 + most.max())) * norm
    del graph
    w.close()
