"""KV page read, the inverse of ``kv_page_write``: gathers cached K and V rows into flat ``[rows][Hkv][D]`` arrays
(swap-out, export of a prefix, inspection). Pages of every ``kv_dtype`` the page write stores; values are rounded to
``dtype`` once and saturate at its largest finite value. No reference counterpart."""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

from . import abi
from .device import Buffer, Device, Stream
from .kv_page_write import Config  # noqa: F401  (one configuration serves both directions)
from .request_page_table import GQAPageTableLayout


@dataclass(frozen=True)
class Shape:
    num_total_token_reads: int
    page_table_layout: GQAPageTableLayout

    def to_c(self) -> abi.KvPageReadShapeC:
        return abi.KvPageReadShapeC(self.num_total_token_reads, self.page_table_layout.to_c())


@dataclass
class Buffers:
    """``flat_k`` / ``flat_v`` are written: row i is the token at position ``flat_token_indices[i]`` of request slot
    ``req_slots[i]``, in any order."""

    pages: Buffer
    flat_k: Buffer
    flat_v: Buffer
    req_slots: Buffer
    flat_token_indices: Buffer
    page_ids: Buffer

    def to_c(self) -> abi.KvPageReadBuffersC:
        return abi.KvPageReadBuffersC(self.pages.ref, self.flat_k.ref, self.flat_v.ref, self.req_slots.ref,
                                      self.flat_token_indices.ref, self.page_ids.ref)


class Compute:
    def __init__(self, device: Device, config: Config):
        handle = C.c_void_p()
        abi.call("kh_kv_page_read_create", device.handle, C.byref(config.to_c()), C.byref(handle))
        self.handle = handle
        self.config = config

    @staticmethod
    def new(device: Device, config: Config) -> "Compute":
        return Compute(device, config)

    def invoke(self, stream: Stream, shape: Shape, buffers: Buffers, num_active_token_reads: int,
               page_table_index: int = 0) -> None:
        """Enqueues the read of the first ``num_active_token_reads`` rows on ``stream``; later rows stay as they are."""
        abi.call("kh_kv_page_read_invoke", self.handle, stream.handle, C.byref(shape.to_c()), C.byref(buffers.to_c()),
                 num_active_token_reads, page_table_index)

    def __del__(self):
        try:
            if self.handle:
                abi.lib().kh_kv_page_read_destroy(self.handle)
                self.handle = None
        except Exception:
            pass
