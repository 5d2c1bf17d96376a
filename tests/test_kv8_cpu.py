"""The 8-bit paged cache without a GPU: what the entry points refuse, and the plain statements that the GPU tests compare with."""
import ctypes as C
import math

import numpy as np
import pytest

from tests import kv8_ref as ref

MAP, APPEND, ATTENTION = 0, 1, 2
AT = 1 << 20  # an address that is only looked at


@pytest.fixture(scope="module")
def lib(built):
    from jitllm_b200 import _lib
    return _lib.load()


def _pages(**changes):
    from jitllm_b200 import _lib
    p = dict(k=AT, v=AT, k_scale=AT, v_scale=AT, block_stride=8 * 16 * 128, scale_stride=8 * 16, blocks=10, block_tokens=16, kv_heads=8, head_dim=128)
    p.update(changes)
    return _lib.JlKv8Pages(**p)


def _args(which, **changes):
    from jitllm_b200 import _lib
    pages = _pages(**{k[6:]: changes.pop(k) for k in list(changes) if k.startswith("pages_")})
    if which == MAP:
        a = dict(held=AT, added=AT, free_blocks=AT, cursor=AT, cursor_out=AT, block_table=AT, lengths=AT, offsets=0, token_slots=0, positions=0,
                 slot_map=AT, result=AT, sequences=3, blocks_per_slot=4, block_tokens=16, free_count=5, capacity=64)
        kind = _lib.JlKv8MapArgs
    elif which == APPEND:
        a = dict(pages=pages, k=AT, v=AT, k_stride=1024, v_stride=1024, slot_map=AT, positions=AT, rope_cos=AT, rope_sin=AT, token_count=0, tokens=3,
                 rope_rows=9, ggml_type=0)
        kind = _lib.JlKv8AppendArgs
    else:
        a = dict(pages=pages, q=AT, out=AT, lse=0, q_stride=4096, out_stride=4096, block_table=AT, kv_slots=0, positions=AT, rope_cos=0, rope_sin=0,
                 token_count=0, rows=3, heads=32, slots=3, blocks_per_slot=4, window=0, rope_rows=0, ggml_type=1, scale=0.1)
        kind = _lib.JlKv8AttentionArgs
    a.update(changes)
    return kind(**a)


def _check(lib, which, args):
    message = C.create_string_buffer(512)
    return lib.jl_debug_kv8_check(which, C.byref(args) if args is not None else None, message, 512), message.value.decode()


@pytest.mark.parametrize("which", [MAP, APPEND, ATTENTION])
def test_the_arguments_that_the_refusals_start_from_pass(lib, which):
    assert _check(lib, which, _args(which)) == (0, "")
    assert _check(lib, which, None)[0] == 1


@pytest.mark.parametrize("changes,status,says", [
    (dict(sequences=0), 6, "sequences"), (dict(sequences=8193), 6, "sequences"), (dict(blocks_per_slot=0), 1, "blocks_per_slot"),
    (dict(block_tokens=0), 1, "block_tokens"), (dict(block_tokens=65537), 1, "block_tokens"), (dict(free_count=-1), 1, "free_count"),
    (dict(capacity=-1), 1, "capacity"), (dict(held=0), 1, "NULL"), (dict(added=0), 1, "NULL"), (dict(cursor=0), 1, "NULL"),
    (dict(cursor_out=0), 1, "NULL"), (dict(block_table=0), 1, "NULL"), (dict(lengths=0), 1, "NULL"), (dict(result=0), 1, "NULL"),
    (dict(free_blocks=0), 1, "free_blocks"), (dict(slot_map=0), 1, "slot_map"), (dict(held=AT + 2), 1, "aligned"),
    (dict(slot_map=AT + 4), 1, "aligned"), (dict(offsets=AT + 1), 1, "aligned")])
def test_map_refuses(lib, changes, status, says):
    rc, message = _check(lib, MAP, _args(MAP, **changes))
    assert rc == status and says in message


def test_map_takes_no_free_blocks_and_no_tokens(lib):
    assert _check(lib, MAP, _args(MAP, free_blocks=0, free_count=0, slot_map=0, capacity=0))[0] == 0


PAGES = [
    (dict(pages_k=0), 1, "NULL"), (dict(pages_v_scale=0), 1, "NULL"), (dict(pages_head_dim=80), 6, "head size 80"), (dict(pages_blocks=0), 1, "blocks"),
    (dict(pages_kv_heads=0), 1, "kv_heads"), (dict(pages_block_tokens=0), 1, "block_tokens"), (dict(pages_block_stride=8 * 16 * 128 - 16), 1, "block_stride"),
    (dict(pages_block_stride=8 * 16 * 128 + 8), 1, "block_stride"), (dict(pages_scale_stride=127), 1, "scale_stride"),
    (dict(pages_block_stride=1 << 62), 1, "64-bit"), (dict(pages_k=AT + 8), 1, "aligned"), (dict(pages_k_scale=AT + 2), 1, "aligned"),
    (dict(ggml_type=8), 6, "GGML type 8"), (dict(rope_cos=AT, rope_sin=0), 1, "both or neither"),
    (dict(rope_cos=AT, rope_sin=AT, rope_rows=0), 1, "rope_rows"), (dict(rope_cos=AT + 4, rope_sin=AT, rope_rows=9), 1, "aligned")]


@pytest.mark.parametrize("changes,status,says", PAGES + [
    (dict(tokens=-1), 1, "tokens"), (dict(tokens=1 << 29), 1, "tokens"), (dict(k=0), 1, "k must not be NULL"), (dict(v=0), 1, "v must not be NULL"),
    (dict(k=AT + 4), 1, "aligned"), (dict(v_stride=1023), 1, "v must"), (dict(k_stride=1000), 1, "k must"), (dict(slot_map=0), 1, "slot_map"),
    (dict(slot_map=AT + 4), 1, "aligned"), (dict(positions=0), 1, "positions"), (dict(ggml_type=1, k_stride=1028), 1, "k must")])
def test_append_refuses(lib, changes, status, says):
    rc, message = _check(lib, APPEND, _args(APPEND, **changes))
    assert rc == status and says in message


@pytest.mark.parametrize("changes,status,says", PAGES + [
    (dict(rows=-1), 1, "rows"), (dict(rows=(1 << 20) + 1), 1, "rows"), (dict(slots=0), 1, "slots"), (dict(blocks_per_slot=0), 1, "blocks_per_slot"),
    (dict(window=-1), 1, "window"), (dict(heads=30), 1, "heads"), (dict(heads=0), 1, "heads"), (dict(heads=32768), 1, "heads"),
    (dict(scale=math.nan), 1, "scale"), (dict(scale=math.inf), 1, "scale"), (dict(q=0), 1, "q must"), (dict(out=0), 1, "out must"),
    (dict(q=AT + 8), 1, "aligned"), (dict(out_stride=4095), 1, "out must"), (dict(q_stride=4092), 1, "q must"), (dict(block_table=0), 1, "block_table"),
    (dict(positions=0), 1, "positions"), (dict(lse=AT + 2), 1, "aligned"), (dict(kv_slots=AT + 1), 1, "aligned")])
def test_attention_refuses(lib, changes, status, says):
    rc, message = _check(lib, ATTENTION, _args(ATTENTION, **changes))
    assert rc == status and says in message


def test_calls_without_a_context_refuse(lib):
    ws = C.c_void_p()
    assert lib.jl_kv8_workspace_create(None, C.byref(ws)) == 1 and not ws
    assert lib.jl_kv8_workspace_free(None, None) == 0
    assert lib.jl_kv8_map(None, None, C.byref(_args(MAP)), None) == 1
    assert lib.jl_kv8_append(None, C.byref(_args(APPEND)), None) == 1
    assert lib.jl_kv8_attention(None, None, C.byref(_args(ATTENTION)), None) == 1
    assert lib.jl_debug_kv8_check(3, None, C.create_string_buffer(8), 8) == 1 and lib.jl_debug_kv8_check(0, None, None, 0) == 1


def test_the_kernels_wait_for_what_is_ahead_before_they_touch_memory():
    """Launched while the kernel ahead still runs, each kernel waits for it before its first access: nothing but its parameters stands in front
    of the wait, in the text."""
    import re
    from pathlib import Path
    from tests.test_kernel_source_rules import CSRC, _code, _function_at
    seen = 0
    for name in ("kv8.cu", "kv8_attention.cu"):
        text = _code(Path(CSRC) / name)
        for m in re.finditer(r"__global__", text):
            body = _function_at(text, m.start())
            in_front = body[:body.index("pdl_wait()")]
            assert not re.search(r"a\.\w+\[|\*reinterpret_cast|__ld|\breturn\b", in_front), name
            seen += 1
    assert seen == 3


def test_plain_map_of_a_small_batch_by_hand():
    """Blocks of 4: a sequence in the middle of a block, one that starts, one that waits, one too long, one beyond the free blocks."""
    table = np.full((5, 3), -1, np.int32)
    table[0, 0] = 9
    table[2, :2] = 7, 8
    slots, pos, place = np.full(40, -5, np.int32), np.full(40, -5, np.int32), np.full(40, -5, np.int64)
    lengths, offsets, cursor, result = ref.map_ref([3, 0, 8, 0, 0], [2, 1, 0, 13, 9], table, np.array([50, 1, 2, 3, 4]), 1, 4, 40, slots, pos, place)
    assert table.tolist() == [[9, 1, -1], [2, -1, -1], [7, 8, -1], [-1, -1, -1], [-1, -1, -1]]
    assert lengths.tolist() == [5, 1, 8, 0, 0] and offsets.tolist() == [0, 2, 3, 3, 16, 25] and cursor == 3
    assert result.tolist() == [25, 2, 2, 5]
    assert place[:4].tolist() == [39, 4, 8, -1] and pos[:4].tolist() == [3, 4, 0, -1] and slots[:4].tolist() == [0, 0, 1, 3]
    assert (place[25:] == -5).all() and (place[3:25] == -1).all()


def test_plain_codes_stand_for_the_values_within_half_a_step():
    x = np.random.default_rng(1).standard_normal((50, 64)) * np.exp(np.random.default_rng(2).standard_normal((50, 1)) * 3)
    codes, scales = ref.quantise(x)
    assert np.abs(codes).max(-1).min() == 127
    assert (np.abs(codes * scales[:, None] - x) <= scales[:, None] * (0.5 + 1e-12)).all()
    codes, scales = ref.quantise(np.array([[0.0, 1e-40], [np.inf, 1.0], [np.nan, 1.0]]))
    assert not codes.any() and scales[0] == 0 and np.isnan(scales[1:]).all()


def test_plain_attention_of_pages_equals_a_softmax_over_rows_in_order():
    rng = np.random.default_rng(3)
    codes, scales = rng.integers(-127, 128, (2, 6, 2, 4, 64)).astype(np.int8), rng.uniform(0.01, 0.02, (2, 6, 2, 4))
    table, q = np.array([[3, 0, 5, -1]]), rng.standard_normal((1, 4, 64))
    out, lse, _ = ref.attention_ref(codes, scales, q, table, None, [9], 0.125, window=7)
    x = (codes * scales[..., None])[:, [3, 0, 5]].transpose(0, 2, 1, 3, 4).reshape(2, 2, 12, 64)[:, :, 3:10]
    for h in range(4):
        s = x[0, h // 2] @ q[0, h] * 0.125
        w = np.exp(s)
        assert np.allclose(out[0, h], w @ x[1, h // 2] / w.sum(), rtol=1e-12) and np.isclose(lse[0, h], np.log(w.sum()), rtol=1e-12)
    out, lse, _ = ref.attention_ref(codes, scales, q, table, None, [-1], 0.125)
    assert not out.any() and (lse == -np.inf).all()
