"""KVCache and RopeCache: the reference's host structs on CUDA memory.

``KVCache`` keeps include/kv_cache.hpp's layout exactly: one buffer of
2 * num_layers * max_seq_len * kv_dim halves; layer l's K at
base + l * 2 * max_seq_len * kv_dim and its V max_seq_len * kv_dim later
(kv_cache.hpp:21-34, :80-82); row t is token t, [t][kv_head][head_dim].
``create_rope_cache`` builds include/rope_cache.hpp:79-105's FP16 cos/sin
tables on the host (b2_fill_rope_tables, FP32 host math) and uploads them.
Device memory comes from torch (plumbing only).

``PagedKVCache`` is the paged form (no counterpart in the reference): a pool of
pages for all layers, a page table, lengths and reference counts on the device,
and the page operations on them.
"""
from __future__ import annotations

import numpy as np

from ._lib import check, lib


class KVCache:
    def __init__(self, num_layers: int, max_seq_len: int, num_kv_heads: int, head_dim: int,
                 device="cuda", buffer=None):
        import torch
        self.num_layers = num_layers
        self.max_seq_len = max_seq_len
        self.num_kv_heads = num_kv_heads
        self.head_dim = head_dim
        self.kv_dim = num_kv_heads * head_dim
        shape = (num_layers, 2, max_seq_len, self.kv_dim)
        if buffer is None:
            buffer = torch.empty(shape, dtype=torch.float16, device=device)
        assert tuple(buffer.shape) == shape and buffer.dtype == torch.float16 and buffer.is_contiguous()
        self.buffer = buffer
        self._cached_len = 0

    def layer_stride(self) -> int:
        return 2 * self.max_seq_len * self.kv_dim

    def get_k_cache(self, layer: int):
        """[max_seq_len, kv_dim] view at base + layer * layer_stride (kv_cache.hpp:21-26)."""
        return self.buffer[layer, 0]

    def get_v_cache(self, layer: int):
        """View at base + layer * layer_stride + max_seq_len * kv_dim (kv_cache.hpp:29-34)."""
        return self.buffer[layer, 1]

    def get_cached_len(self) -> int:
        return self._cached_len

    def set_cached_len(self, cached_len: int) -> None:
        if cached_len > self.max_seq_len:  # kv_cache.hpp:40-45
            raise IndexError(f"KV cache capacity exceeded: requested {cached_len} tokens, "
                             f"capacity {self.max_seq_len}")
        self._cached_len = cached_len

    def reset_cache(self) -> None:
        self._cached_len = 0


class PagedKVCache:
    """Pages of page_size tokens for num_layers layers' K and V, shared by up to
    max_seqs sequences of at most max_pages_per_seq pages each.

    The state lies on the device (page_table, seq_len, ref_count), and so do the
    operations' arguments: contiguous int32 tensors of table rows, lengths and
    counts on the same device (pos and the arrays after the first may be longer). The
    operations are launches (no synchronisation, capturable); ``check`` waits for the
    last truncate, fork, extend or compact and reads its status. Calls are ordered on one stream, or by the caller.
    """

    def __init__(self, num_layers: int, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int,
                 max_seqs: int, max_pages_per_seq: int, device="cuda"):
        import torch
        self.num_layers, self.num_pages, self.page_size = num_layers, num_pages, page_size
        self.num_kv_heads, self.head_dim = num_kv_heads, head_dim
        self.kv_dim = num_kv_heads * head_dim
        self.max_seqs, self.max_pages_per_seq = max_seqs, max_pages_per_seq
        # plane 2 l: layer l's K pages, plane 2 l + 1: its V pages
        self.buffer = torch.empty((2 * num_layers, num_pages, page_size, self.kv_dim), dtype=torch.float16,
                                  device=device)

        def ints(shape, value):
            return torch.full(shape, value, dtype=torch.int32, device=device)

        self.page_table = ints((max_seqs, max_pages_per_seq), -1)
        self.seq_len = ints((max_seqs,), 0)
        self.ref_count = ints((num_pages,), 0)
        self.status = ints((2,), 0)
        self._ws_bytes = int(lib().b2_kv_pages_workspace_bytes(num_pages))
        if self._ws_bytes == 0:
            raise ValueError(f"{num_pages} pages: 1 to 2**21 are possible")
        self._ws = torch.zeros(self._ws_bytes, dtype=torch.uint8, device=device)
        self._device = self._ws.device
        self._stream = None      # the last operation's
        self._streams = set()    # those other than torch's own that have used the cache
        if self._ws.is_cuda:   # written before a stream that does not wait for torch's uses them
            torch.cuda.current_stream(self._device).synchronize()

    def get_k_pages(self, layer: int):
        """[num_pages, page_size, kv_dim] K pages of a layer."""
        return self.buffer[2 * layer]

    def get_v_pages(self, layer: int):
        return self.buffer[2 * layer + 1]

    def pages(self, layer: int):
        """The cache arguments of the paged launchers: from d_k_pages to table_rows."""
        return (self.get_k_pages(layer), self.get_v_pages(layer), 0, self.num_pages, self.page_size, self.page_table,
                self.max_pages_per_seq, self.max_seqs)

    def _pool(self):
        return self.buffer, 2 * self.num_layers, 0, self.num_pages, 0, self.page_size * self.kv_dim

    def _table(self):
        return self.page_table, self.max_pages_per_seq, self.max_seqs, self.page_size

    def _items(self, stream, *arrays):
        """Items of a call: elements of its first array. The others hold as many
        at least, or the kernels would read past their ends."""
        import torch
        n, device = arrays[0].numel(), self._device
        for t in arrays:
            if t is None:
                continue
            if t.dtype != torch.int32 or not t.is_contiguous() or t.numel() < n or t.device != device:
                raise ValueError(f"expected {n} contiguous int32 on {device}; got {t.numel()} "
                                 f"{'' if t.is_contiguous() else 'strided '}{t.dtype} on {t.device}")
        self._current()
        self._used_on(stream, *arrays)
        return n

    def _used_on(self, stream, *arrays):
        """The memory of arrays, and of the cache, that die before a stream other than torch's own is done with them
        is not given out again (what a graph holds lives as long as the graph: its maker sees to that)."""
        import torch
        handle = self._handle(stream)
        # (the raw handle: torch.cuda.current_stream takes as long as all the rest of a call)
        if not self._ws.is_cuda or handle == torch._C._cuda_getCurrentRawStream(self._device.index):
            return
        with torch.cuda.stream(self._torch_stream(stream)):
            if torch.cuda.is_current_stream_capturing():
                return
            if handle not in self._streams:
                self._streams.add(handle)
                arrays += (self.buffer, self.page_table, self.seq_len, self.ref_count, self.status, self._ws)
            for t in arrays:
                if t is not None:
                    t.record_stream(torch.cuda.current_stream(self._device))

    @staticmethod
    def _handle(stream):
        return (stream if isinstance(stream, int) else stream.cuda_stream) if stream is not None else 0

    def _torch_stream(self, stream):
        import torch
        device, handle = self._device, self._handle(stream)
        return torch.cuda.ExternalStream(handle, device=device) if handle else torch.cuda.default_stream(device)

    def _current(self):
        import torch
        device = self._device
        if device.type == "cuda" and device.index != torch.cuda.current_device():
            raise ValueError(f"the cache lies on {device}, which is not the current device")

    def _work(self, stream):
        return self.status, self._ws, self._ws_bytes, stream

    def _launched(self, n, stream):
        """An operation of n items went to this stream (one without items goes nowhere)."""
        if n:
            self._stream = stream

    def extend(self, seqs, new_tokens, pos=None, stream=None):
        """Room for new_tokens[i] more tokens of sequence seqs[i]; pos[i] = its first new position."""
        from .kernels import launch_kv_pages_extend
        n = self._items(stream, seqs, new_tokens, pos)
        launch_kv_pages_extend(*self._pool(), *self._table(), self.seq_len, self.ref_count, seqs, new_tokens,
                               n, pos, *self._work(stream))
        self._launched(n, stream)

    def truncate(self, seqs, new_len=None, stream=None):
        """Sequence seqs[i] keeps its first new_len[i] tokens (None: it is freed)."""
        from .kernels import launch_kv_pages_truncate
        n = self._items(stream, seqs, new_len)
        launch_kv_pages_truncate(*self._table(), self.num_pages, self.seq_len, self.ref_count, seqs, new_len,
                                 n, *self._work(stream))
        self._launched(n, stream)

    def fork(self, parents, children, fork_len=None, stream=None):
        """Empty sequence children[i] shares the first fork_len[i] tokens (None: all) of parents[i]."""
        from .kernels import launch_kv_pages_fork
        n = self._items(stream, parents, children, fork_len)
        launch_kv_pages_fork(*self._table(), self.num_pages, self.seq_len, self.ref_count, parents, children,
                             fork_len, n, *self._work(stream))
        self._launched(n, stream)

    def compact(self, stream=None):
        """Brings the live pages together at the low numbers; status[1] = how many they are."""
        from .kernels import launch_kv_pages_compact
        self._current()
        self._used_on(stream)
        launch_kv_pages_compact(*self._pool(), self.page_table, *self._table(), self.seq_len, self.ref_count,
                                self.ref_count, *self._work(stream))
        self._launched(1, stream)

    def copy_pages(self, src, dst, stream=None):
        """Contents of page dst[i] = those of page src[i], every layer."""
        from .kernels import launch_kv_pages_copy
        launch_kv_pages_copy(*self._pool(), src, dst, self._items(stream, src, dst), stream)

    def check(self, stream=None):
        """Raises if the last truncate, fork or extend was refused; returns status[1] (a compact's: the live pages).
        Waits for the stream that the last of these was launched on, or for ``stream``: the one that a graph of
        captured operations runs on. A call without items is none."""
        stream = self._stream if stream is None else stream
        if self.page_table.is_cuda:
            self._torch_stream(stream).synchronize()
        code, count = self.status.tolist()
        if code == 1:
            raise MemoryError(f"too few free pages: the call takes {count}")
        if code != 0:
            raise ValueError("bad item: a row outside the table, a sequence named twice, a length out of range, a "
                             "child that is not empty, or a partly filled last page that is outside the pool or "
                             "without a reference")
        return count


def rope_tables_host(max_seq_len: int, head_dim: int, rope_theta: float):
    """FP16 cos/sin [max_seq_len, head_dim/2] as numpy float16 (rope_cache.hpp:49-76)."""
    half = head_dim // 2
    cos = np.zeros((max_seq_len, half), np.uint16)
    sin = np.zeros((max_seq_len, half), np.uint16)
    check(lib().b2_fill_rope_tables(max_seq_len, head_dim, float(rope_theta),
                                    cos.ctypes.data, sin.ctypes.data), "fill_rope_tables")
    return cos.view(np.float16), sin.view(np.float16)


class RopeCache:
    def __init__(self, d_cos, d_sin):
        self.d_cos = d_cos
        self.d_sin = d_sin


def create_rope_cache(max_seq_len: int, head_dim: int, rope_theta: float, device="cuda") -> RopeCache:
    import torch
    cos, sin = rope_tables_host(max_seq_len, head_dim, rope_theta)
    return RopeCache(torch.from_numpy(cos).to(device), torch.from_numpy(sin).to(device))
