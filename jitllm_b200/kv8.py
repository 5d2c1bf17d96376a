"""The 8-bit paged key/value cache: block maps from sequence lengths, append, single-token attention (jl_kv8_* of
include/jitllm_b200.h, which describes every field).

Like DeviceMatrix.matmul_dev these take device addresses (integers: Device.alloc, or the data_ptr() of a tensor on that GPU),
not arrays. A call is an object made once, with its buffers, and launched at every step; `launch(stream)` enqueues it on a
cudaStream_t given as an integer (0: the default stream), or on the context's own stream without one, and does not wait. The
buffers have to outlive the launches. Arguments are checked by the library at each launch: ValueError as everywhere."""
from __future__ import annotations

import ctypes as C
from typing import Optional

from . import _lib
from .api import Device, GGMLType, IllegalStateError


def _struct(kind, *values):
    """The argument structure. ctypes would cut a number that its field has no room for."""
    for (name, field), value in zip(kind._fields_, values):
        if field in (C.c_int32, C.c_int64, C.c_void_p) and value is not None:
            bits = 8 * C.sizeof(field)
            if not (0 if field is C.c_void_p else -(1 << bits - 1)) <= value < 1 << (bits if field is C.c_void_p else bits - 1):
                raise ValueError(f"{name} = {value} does not fit into {bits} bits")
    return kind(*values)


class Kv8Workspace:
    """Partial results and arrival counters of jl_kv8_map and jl_kv8_attention. Calls with one workspace must not overlap on
    the GPU: one for each stream (or captured graph) that runs beside others. Closed with the device at the latest: keep it
    until no call with it is under way and no graph holds one."""

    def __init__(self, dev: Device):
        self.dev = dev
        h = C.c_void_p()
        dev._check(dev._lib.jl_kv8_workspace_create(dev.handle, C.byref(h)))
        self._h = h

    @property
    def handle(self):
        if self._h is None or self.dev._h is None:
            raise IllegalStateError("GPUL-LIFE-001: this workspace is closed")
        return self._h

    def close(self) -> None:
        if self._h is not None and self.dev._h is not None:
            self.dev._lib.jl_kv8_workspace_free(self.dev.handle, self._h)
        self._h = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()


class Kv8Pages:
    """Pages of int8 codes [blocks][kvHeads][blockSizeTokens][headSize] and binary32 scales [blocks][kvHeads][blockSizeTokens],
    keys and values, in device memory of the caller. blockStride (bytes) and scaleStride (floats) from one block to the next
    default to blocks without gaps."""

    def __init__(self, dev: Device, k: int, v: int, kScale: int, vScale: int, *, blocks: int, blockSizeTokens: int,
                 kvHeads: int, headSize: int, blockStride: Optional[int] = None, scaleStride: Optional[int] = None):
        self.dev = dev
        rows = kvHeads * blockSizeTokens
        self.struct = _struct(
            _lib.JlKv8Pages, k, v, kScale, vScale, rows * headSize if blockStride is None else blockStride,
            rows if scaleStride is None else scaleStride, blocks, blockSizeTokens, kvHeads, headSize)

    def bytesPerBlock(self) -> int:
        p = self.struct
        return 2 * p.kv_heads * p.block_tokens * (p.head_dim + 4)


class _Call:
    """An entry point with its arguments."""

    def __init__(self, dev: Device, entry: str, args: C.Structure, workspace: Optional[Kv8Workspace] = None):
        self.dev, self.args, self.workspace = dev, args, workspace
        self._entry = getattr(dev._lib, entry)
        self._ref = C.byref(args)

    def launch(self, stream: Optional[int] = None) -> None:
        dev, ws = self.dev, self.workspace
        h = dev._h
        if h is None or (ws is not None and (ws._h is None or ws.dev._h is None)):
            raise IllegalStateError("GPUL-LIFE-001: the device context or the workspace is closed")
        if stream is None:
            stream = dev._lib.jl_stream(h)
        rc = self._entry(h, self._ref, stream) if ws is None else self._entry(h, ws._h, self._ref, stream)
        if rc != 0:
            dev._check(rc)


class Kv8Map(_Call):
    """Block table and slot map from the sequences' lengths: jl_kv8_map."""

    def __init__(self, workspace: Kv8Workspace, *, held: int, added: int, sequences: int, blockTable: int, blocksPerSlot: int,
                 blockSizeTokens: int, freeBlocks: int, freeCount: int, cursor: int, cursorOut: int, lengths: int,
                 slotMap: int, capacity: int, result: int, offsets: int = 0, tokenSlots: int = 0, positions: int = 0):
        super().__init__(workspace.dev, "jl_kv8_map", _struct(
            _lib.JlKv8MapArgs, held, added, freeBlocks, cursor, cursorOut, blockTable, lengths, offsets, tokenSlots, positions, slotMap, result,
            sequences, blocksPerSlot, blockSizeTokens, freeCount, capacity), workspace)


class Kv8Append(_Call):
    """Keys and values of new tokens to their places in the pages: jl_kv8_append. Strides in elements, by default those of
    rows without gaps; rotation tables as of B200Model.uploadRope."""

    def __init__(self, pages: Kv8Pages, k: int, v: int, ggml_type: GGMLType, *, tokens: int, slotMap: int,
                 keyStride: Optional[int] = None, valueStride: Optional[int] = None, positions: int = 0, ropeCos: int = 0,
                 ropeSin: int = 0, ropeRows: int = 0, tokenCount: int = 0):
        row = pages.struct.kv_heads * pages.struct.head_dim
        super().__init__(pages.dev, "jl_kv8_append", _struct(
            _lib.JlKv8AppendArgs, pages.struct, k, v, row if keyStride is None else keyStride, row if valueStride is None else valueStride, slotMap,
            positions, ropeCos, ropeSin, tokenCount, tokens, ropeRows, int(ggml_type)))


class Kv8Attention(_Call):
    """Attention of single tokens over the pages: jl_kv8_attention. Strides in elements, by default those of rows without
    gaps; scale is what q.k is multiplied by, by default 1 / sqrt(headSize)."""

    def __init__(self, pages: Kv8Pages, workspace: Kv8Workspace, q: int, out: int, ggml_type: GGMLType, *, rows: int, heads: int,
                 blockTable: int, slots: int, blocksPerSlot: int, positions: int, kvSlots: int = 0, lse: int = 0,
                 queryStride: Optional[int] = None, outStride: Optional[int] = None, window: int = 0,
                 scale: Optional[float] = None, ropeCos: int = 0, ropeSin: int = 0, ropeRows: int = 0, tokenCount: int = 0):
        d = pages.struct.head_dim
        row = heads * d
        super().__init__(pages.dev, "jl_kv8_attention", _struct(
            _lib.JlKv8AttentionArgs, pages.struct, q, out, lse, row if queryStride is None else queryStride, row if outStride is None else outStride,
            blockTable, kvSlots, positions, ropeCos, ropeSin, tokenCount, rows, heads, slots, blocksPerSlot, window, ropeRows,
            int(ggml_type), d ** -0.5 if scale is None else scale), workspace)
