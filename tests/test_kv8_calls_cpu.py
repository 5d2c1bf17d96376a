"""The Python calls of the 8-bit paged cache without a GPU, beside tests/test_kv8_cpu.py."""
import re
from pathlib import Path
from types import SimpleNamespace

import pytest

import jitllm_b200 as jl
from tests.test_kernel_source_rules import CSRC, _code, _function_at
from tests.test_kv8_cpu import ATTENTION, _args, _check, lib  # noqa: F401

AT = 1 << 20


def _pages(dev, **changes):
    return jl.Kv8Pages(dev, **{**dict(k=AT, v=AT, kScale=AT, vScale=AT, blocks=10, blockSizeTokens=16, kvHeads=8, headSize=128), **changes})


def _calls(lib, name, **changes):  # noqa: F811
    dev = SimpleNamespace(_lib=lib)
    if name == "pages":
        return _pages(dev, **changes).struct
    if name == "map":
        kw = dict(held=AT, added=AT, sequences=3, blockTable=AT, blocksPerSlot=4, blockSizeTokens=16, freeBlocks=AT, freeCount=5, cursor=AT, cursorOut=AT,
                  lengths=AT, slotMap=AT, capacity=64, result=AT)
        return jl.Kv8Map(SimpleNamespace(dev=dev), **{**kw, **changes}).args
    if name == "append":
        kw = dict(k=AT, v=AT, ggml_type=jl.GGMLType.F32, tokens=3, slotMap=AT)
        return jl.Kv8Append(_pages(dev), **{**kw, **changes}).args
    kw = dict(q=AT, out=AT, ggml_type=jl.GGMLType.F32, rows=3, heads=32, blockTable=AT, slots=3, blocksPerSlot=4, positions=AT)
    return jl.Kv8Attention(_pages(dev), None, **{**kw, **changes}).args


@pytest.mark.parametrize("name,changes,field", [
    ("pages", dict(blocks=2 ** 32 + 10), "blocks"), ("pages", dict(blockStride=2 ** 63), "block_stride"), ("pages", dict(k=-16), "k"),
    ("pages", dict(vScale=2 ** 64), "v_scale"), ("map", dict(sequences=2 ** 32 + 3), "sequences"), ("map", dict(capacity=2 ** 32 + 64), "capacity"),
    ("map", dict(freeCount=2 ** 31), "free_count"), ("append", dict(tokens=2 ** 32 + 1), "tokens"), ("append", dict(keyStride=2 ** 64 + 1024), "k_stride"),
    ("append", dict(ropeRows=-2 ** 31 - 1), "rope_rows"), ("attention", dict(rows=2 ** 32), "rows"), ("attention", dict(window=2 ** 32 + 1000), "window"),
    ("attention", dict(blocksPerSlot=2 ** 40), "blocks_per_slot"), ("attention", dict(queryStride=-2 ** 63 - 1), "q_stride")])
def test_numbers_that_a_field_has_no_room_for_are_refused(lib, name, changes, field):  # noqa: F811
    """ctypes would cut them: a window of 2^32 + 1000 tokens would be one of 1000."""
    with pytest.raises(ValueError, match=f"^{field} = "):
        _calls(lib, name, **changes)


@pytest.mark.parametrize("name,changes", [("pages", {}), ("map", dict(capacity=2 ** 31 - 1)), ("append", dict(tokenCount=2 ** 64 - 4)), ("attention", dict(window=2 ** 31 - 1, lse=None))])
def test_numbers_that_fit_arrive(lib, name, changes):  # noqa: F811
    args = _calls(lib, name, **changes)
    for key, value in changes.items():
        assert getattr(args, {"tokenCount": "token_count"}.get(key, key)) == value


def test_the_largest_number_of_rows(lib):  # noqa: F811
    assert _check(lib, ATTENTION, _args(ATTENTION, rows=1 << 16)) == (0, "")
    rc, message = _check(lib, ATTENTION, _args(ATTENTION, rows=(1 << 16) + 1))
    assert rc == 1 and "rows" in message


def test_bytes_of_a_block_of_pages(lib):  # noqa: F811
    """Codes and scales of keys and values, as KvStorage.bytesPerBlock() of the model's own store; gaps between blocks are the caller's."""
    pages = _pages(SimpleNamespace(_lib=lib), blockStride=8 * 16 * 128 + 64, scaleStride=200)
    assert pages.bytesPerBlock() == 2 * 8 * 16 * (128 + 4)


@pytest.mark.parametrize("name,kernels", [("kv8.cu", 2), ("kv8_attention.cu", 1)])
def test_in_front_of_the_wait_there_are_declarations_only(name, kernels):
    """A kernel that is launched while the one ahead still runs may not touch memory before pdl_wait(): what stands in front of it are types,
    shared arrays, and numbers made of the thread's and the block's indexes and of the parameters."""
    text = _code(Path(CSRC) / name)
    found = 0
    for m in re.finditer(r"__global__", text):
        body = _function_at(text, m.start())
        in_front = body[body.index("{") + 1:body.index("pdl_wait()")]
        found += 1
        for statement in (x.strip() for x in in_front.split(";")):
            statement = " ".join(statement.split())
            assert (re.fullmatch(r"(using .*|constexpr [\w ]+ = .*|pdl_launch_dependents\(\)|)", statement)
                    or re.fullmatch(r"(extern )?__shared__ [^=]*", statement)
                    or re.fullmatch(r"const \w+ &a = p\.a", statement)
                    or re.fullmatch(r"const (int|uint32_t) (\w+ = [\w.%<>&+\- ]+(, )?)+", statement)), statement
    assert found == kernels
