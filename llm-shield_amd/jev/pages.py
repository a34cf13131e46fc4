"""The paged 8-bit KV cache over libjev's jev_pages_* entry points: one pool of pages
in HBM that many requests share, planned on the device (include/jev.h has the rules)."""
from __future__ import annotations

import ctypes

from . import _lib as L
from .model import ModelConfig, _i32


class KvPages:
    """A pool of `n_pages` pages of `page_tokens` tokens for up to `max_requests` requests.

    The *_device calls take device pointers (integers) and only enqueue on the handle's stream."""

    def __init__(self, config: ModelConfig, n_pages: int, page_tokens: int = 16, max_requests: int = 64,
                 max_context: int = 4096, max_tokens: int = 4096, rope_half: bool = False, device: int = 0):
        self._h = ctypes.c_void_p()
        self._lib = L.lib()
        self.config, self.n_pages, self.page_tokens = config, n_pages, page_tokens
        self.max_requests, self.max_context, self.max_tokens = max_requests, max_context, max_tokens
        c = L.PagesConfig(n_pages, page_tokens, max_requests, max_context, max_tokens, int(rope_half))
        L.check(self._lib.jev_pages_create(ctypes.byref(config.to_c()), ctypes.byref(c), device, ctypes.byref(self._h)))

    def close(self) -> None:
        if self._h:
            self._lib.jev_pages_destroy(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    @property
    def handle(self) -> ctypes.c_void_p:
        return self._h

    @property
    def stream(self) -> int:
        """The handle's HIP stream (for graph capture or ordering by the caller)."""
        return int(self._lib.jev_pages_stream(self._h) or 0)

    def plan_device(self, request: int, past: int, fresh: int, n_requests: int, n_tokens: int, table: int = 0, slot: int = 0,
                    position: int = 0, row: int = 0, start: int = 0) -> None:
        """A step's bookkeeping: batch row b keeps past[b] tokens of request[b] (past 0: all) and adds fresh[b]."""
        L.check(self._lib.jev_pages_plan_device(self._h, request, past, fresh, n_requests, n_tokens, table, slot, position, row, start))

    def store_device(self, layer: int, q: int, q_ld: int, k: int, v: int, kv_ld: int, q_out: int) -> None:
        """Rotates the planned tokens' q into q_out and stores their k (rotated) and v; 0 for q and q_out, or k and v: not these."""
        L.check(self._lib.jev_pages_store_device(self._h, layer, q, q_ld, k, v, kv_ld, q_out))

    def attend_device(self, layer: int, q: int, out: int) -> None:
        """The planned tokens' attention over their requests' pages."""
        L.check(self._lib.jev_pages_attend_device(self._h, layer, q, out))

    def read_device(self, layer: int, slot: int, n: int, k: int, v: int) -> None:
        """The values stored at n slots."""
        L.check(self._lib.jev_pages_read_device(self._h, layer, slot, n, k, v))

    def release(self, requests) -> None:
        """Gives back all pages of `requests` (host integers)."""
        ids = _i32(list(requests))
        L.check(self._lib.jev_pages_release(self._h, ids.ctypes.data_as(ctypes.POINTER(ctypes.c_int32)), len(ids)))

    def sync(self) -> None:
        """Waits for the handle's work; raises if the last plan was refused."""
        L.check(self._lib.jev_pages_sync(self._h))
