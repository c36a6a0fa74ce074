"""A paged bank cache: sequences share the pages of equal banks until one writes.

The reference counts what a copy-on-write cache of its layers would hold
(APPENDIX.md:511-584; ``written_banks`` and ``cow_worst_case_bytes`` here) and
serves from dense caches.  ``BankPages`` is such a cache.  One pool holds a page
[H, S, v] for each bank that differs between its holders; ``table[layer,
sequence, bank]`` names a bank's page and ``references`` counts the table entries
of each page.  Forked sequences (beams, samples of one prompt) share every page,
a prompt shares the banks it did not write with the initial state, and a decode
step gives a bank a page of its own when it first writes it: the decode kernel
reads the shared page and stores to the new one.

Every call enqueues its kernels on the current stream of the pool's device and
returns without synchronising; calls on one cache from several streams are the
caller's to order.  All of them but ``check`` may be captured in a HIP graph,
whose replays need the handle kept alive.
New pages are the lowest-numbered free ones in the order of the requests, so
tables do not change from run to run.
"""

from __future__ import annotations

import ctypes

import torch
from torch import Tensor

from . import _lib, ops

MAX_SEQUENCES = 512
MAX_SELECTED = 16  # written, and read, banks of a token


class BankPages:
    """A pool of ``pages`` bank pages for ``layers`` x ``sequences`` x ``banks`` banks.

    Every sequence starts without pages.  layers * sequences * banks pages are
    the most that calls leave in use; a decode step needs its new pages before
    those that it abandons are free, one for every two written banks at most, so
    sequences * KW / 2 more always suffice.  With fewer, ``check`` tells whether a
    call found none left (the bank then kept its old content, or no page in
    ``load``)."""

    def __init__(self, sequences: int, pages: int, *, banks: int, heads: int, bank_size: int, head_width: int,
                 layers: int = 1, dtype: torch.dtype = torch.bfloat16, device='cuda') -> None:
        sizes = dict(sequences=sequences, pages=pages, banks=banks, heads=heads, bank_size=bank_size,
                     head_width=head_width, layers=layers)
        bad = [name for name, value in sizes.items() if type(value) is not int or value < 1]
        if bad:
            raise ValueError(f'BankPages needs positive {", ".join(bad)}')
        if dtype not in (torch.float32, torch.bfloat16):
            raise ValueError('cache dtype must be FP32 or BF16')
        device = torch.device(device)
        if device.type != 'cuda':
            raise ValueError('BankPages needs a ROCm device')
        self._adopt(torch.zeros(pages, heads, bank_size, head_width, dtype=dtype, device=device),
                    torch.full((layers, sequences, banks), -1, dtype=torch.int32, device=device),
                    torch.zeros(pages, dtype=torch.int32, device=device))

    @classmethod
    def over(cls, pool: Tensor, table: Tensor, references: Tensor) -> 'BankPages':
        """A cache over existing tensors, used in place: pool [P, H, S, v] FP32
        or BF16, table [layers, sequences, banks] int32 (pages of the pool, or
        -1 throughout a sequence), references [P] int32, the number of table
        entries of each page.  The tensors have to agree with each other, and a
        page may be an entry of one layer and bank only.  From then on table and
        references change through this handle alone, which keeps a map of the
        free pages beside them: behind a change of the caller's own (a restored
        snapshot, for instance) a new handle is made over the tensors."""
        if pool.ndim != 4 or table.ndim != 3 or references.shape != pool.shape[:1] or 0 in (*pool.shape, *table.shape):
            raise ValueError('pool must be [pages, heads, bank_size, head_width], table [layers, sequences, banks] and '
                             'references [pages]')
        if pool.dtype not in (torch.float32, torch.bfloat16) or torch.int32 not in {table.dtype, references.dtype}:
            raise ValueError('pool must be FP32 or BF16, table and references int32')
        if table.dtype != references.dtype or not all(t.is_contiguous() for t in (pool, table, references)):
            raise ValueError('pool, table and references must be contiguous, table and references int32')
        ops._require_gpu(pool, table, references)
        if pool.data_ptr() % 16:
            raise ValueError('the pool must be 16-byte aligned')
        self = cls.__new__(cls)
        self._adopt(pool, table, references)
        return self

    def _adopt(self, pool: Tensor, table: Tensor, references: Tensor) -> None:
        self.pool, self.table, self.references = pool, table, references
        self.layers, self.sequences, self.banks = table.shape
        if self.sequences > MAX_SEQUENCES:
            raise NotImplementedError(f'BankPages takes at most {MAX_SEQUENCES} sequences')
        self.pages, self.heads, self.bank_size, self.head_width = pool.shape
        self.dtype, self.device = pool.dtype, pool.device
        self._index = pool.get_device()
        # one bit a page: set where nothing references it, 64 pages a word
        free = torch.zeros((self.pages + 63) // 64 * 64, dtype=torch.int64, device=self.device)
        free[:self.pages] = references == 0
        self.free_bits = (free.view(-1, 64) << torch.arange(64, device=self.device)).sum(-1)
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        args = self._args = _lib.Pages()
        args.pool, args.table, args.references, args.free_bits, args.status = (
            t.data_ptr() for t in (pool, table, references, self.free_bits, self.status))
        args.pages, args.layers, args.sequences, args.banks = self.pages, *table.shape
        args.heads, args.bank_size, args.head_width = self.heads, self.bank_size, self.head_width
        args.dtype = ops._dtype_code(pool.dtype)
        self._ref = ctypes.byref(args)
        step = self._step = _lib.DecodeArgs()  # the fields that every step shares
        step.heads, step.bank_size, step.head_width, step.bank_count = (self.heads, self.bank_size, self.head_width,
                                                                        self.banks)
        step.state_dtype = args.dtype
        self._step_ref = ctypes.byref(step)
        # the tables of one step, the handle's own: calls on one cache are ordered, so nothing else uses them meanwhile
        nbytes = _lib.library().bdm_pages_decode_workspace_size(self._ref, MAX_SELECTED, MAX_SELECTED)
        self._tables = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        self._library = _lib.library()
        self._streams = {ops._stream(self.device)}  # the one that the tensors belong to

    def _on_stream(self) -> int:
        """The current stream.  The tensors are recorded on each but their own that a call uses: their memory is not
        given back while one of them still runs, also where the handle is dropped before."""
        stream = ops._stream(self.device)
        if stream not in self._streams:
            current = torch.cuda.current_stream(self.device)
            for t in (self.pool, self.table, self.references, self.free_bits, self.status, self._tables):
                t.record_stream(current)
            self._streams.add(stream)
        return stream

    # -- bookkeeping ------------------------------------------------------------------
    def used(self) -> Tensor:
        """The number of pages in use, a device scalar."""
        self._on_stream()
        return (self.references > 0).sum()

    def check(self) -> None:
        """Raises if a call since the last check found no free page.
        Synchronises the host."""
        self._on_stream()
        if int(self.status):
            self.status.zero_()
            raise RuntimeError(f'BankPages: no free page was left of {self.pages}')

    def _rows(self, sequences) -> list[int]:
        rows = [sequences] if isinstance(sequences, int) else [int(i) for i in sequences]
        if rows and (min(rows) < 0 or max(rows) >= self.sequences or len(set(rows)) != len(rows)):
            raise ValueError(f'sequences must be distinct and below {self.sequences}')
        return rows

    def _layer(self, layer: int) -> int:
        if not 0 <= layer < self.layers:
            raise ValueError(f'layer must be 0 to {self.layers - 1}')
        return int(layer)

    def _call(self, name: str, *arguments) -> None:
        device, stream = self.device, self._on_stream()
        if device.index == torch.cuda.current_device():
            status = getattr(self._library, name)(self._ref, *arguments, stream)
        else:
            with torch.cuda.device(device):
                status = getattr(self._library, name)(self._ref, *arguments, stream)
        if status:
            _lib.check(status, name)

    # -- copying, forking, compacting and freeing -------------------------------------
    def load(self, layer: int, sequences, states: Tensor, base: int | None = None) -> None:
        """Dense states [n, banks, heads, bank_size, head_width] become the banks
        of the n ``sequences`` (Python ints) in ``layer``; what these held is
        dropped first.  A bank that equals the ``base`` sequence's bit for bit
        shares its page.  [n, banks, bank_size, width] caches of one head are
        taken too."""
        rows, layer = self._rows(sequences), self._layer(layer)
        shape = (len(rows), self.banks, self.heads, self.bank_size, self.head_width)
        if states.ndim == 4 and self.heads == 1:
            states = states.unsqueeze(2)
        if tuple(states.shape) != shape or states.dtype != self.dtype:
            raise ValueError(f'states must be {self.dtype} {shape}')
        if base is not None and (not 0 <= base < self.sequences or base in rows):
            raise ValueError('base must be another sequence')
        if states.device != self.device:
            raise ValueError('all tensors must be on the device of the pages')
        states = states.contiguous()
        # pages that the sequences leave can be given to the banks of others, ahead of a read of them
        if self.pool.data_ptr() < states.data_ptr() + states.nbytes and (
                states.data_ptr() < self.pool.data_ptr() + self.pool.nbytes):
            states = states.clone()
        nbytes = _lib.library().bdm_pages_load_workspace_size(self._ref, len(rows))
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        self._call('bdm_pages_load', layer, (ctypes.c_int32 * len(rows))(*rows), len(rows),
                   -1 if base is None else int(base), states.data_ptr(), workspace.data_ptr(), nbytes)

    def dense(self, layer: int, sequences) -> Tensor:
        """The banks of ``sequences`` in ``layer`` as dense states [n, banks,
        heads, bank_size, head_width]: zeros for a sequence without pages."""
        rows, layer = self._rows(sequences), self._layer(layer)
        out = torch.empty(len(rows), self.banks, self.heads, self.bank_size, self.head_width, dtype=self.dtype,
                          device=self.device)
        self._call('bdm_pages_dense', layer, (ctypes.c_int32 * len(rows))(*rows), len(rows), out.data_ptr())
        return out

    def fork(self, parents: Tensor) -> None:
        """Sequence i continues sequence ``parents[i]``, in every layer: int64,
        entries for the first sequences (the others stay).  A negative entry
        releases the sequence's pages, one behind the last sequence counts as the
        last.  Tables and reference counts change, no
        page is copied."""
        if parents.dtype != torch.int64 or not 1 <= parents.numel() <= self.sequences:
            raise ValueError(f'parents must be int64, for 1 to {self.sequences} sequences')
        if parents.device != self.device:
            raise ValueError('all tensors must be on the device of the pages')
        parents = parents.contiguous()
        self._call('bdm_pages_fork', parents.data_ptr(), None, parents.numel())

    def release(self, sequences) -> None:
        """Drops the pages of ``sequences`` (Python ints) in every layer."""
        rows = self._rows(sequences)
        self._call('bdm_pages_fork', None, (ctypes.c_int32 * len(rows))(*rows), len(rows))

    def compact(self) -> None:
        """Moves the used pages to the front of the pool: behind it, the first
        ``used()`` pages are those in use."""
        nbytes = _lib.library().bdm_pages_compact_workspace_size(self._ref)
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        self._call('bdm_pages_compact', workspace.data_ptr(), nbytes)

    # -- the decode step ----------------------------------------------------------------
    def decode(self, layer: int, q, k, v, g, b, w, wi, ww, ri, rw, *, scale: float, routed_decay: bool) -> Tensor:
        """One token for each of the first N sequences over its pages of ``layer``:
        the step of ``ops.decode_step``, q, k, g, b [N, H, S], v, w [N, H, v], wi,
        ww [N, KW], ri, rw [N, KR].  Returns y [N, H*v].  A bank that is written while other sequences hold its page too moves to a
        new page.  Products with the route weights and the sum over the read
        banks are FP32 here and y is rounded once: with FP32 controllers the
        result is ``decode_step``'s bit for bit, with BF16 ones it is nearer to
        the exact one.  Sequences without pages give 0 and stay without."""
        # each look at a tensor's attribute is 0.1 to 0.3 us of the host, which a step of few sequences waits for: every
        # one is asked for once
        layer, device, dtype, shape = self._layer(layer), self.device, q.dtype, q.shape
        n, heads, s, width = shape[0] if shape else 0, self.heads, self.bank_size, self.head_width
        if not 1 <= n <= self.sequences:
            raise ValueError(f'decode takes 1 to {self.sequences} sequences')
        rows, columns = (n, heads, s), (n, heads, width)
        if (shape != rows or k.shape != rows or g.shape != rows or b.shape != rows or v.shape != columns
                or w.shape != columns):
            raise ValueError(f'q, k, g, b must be {rows} and v, w {columns}')
        writes, reads = wi.shape, ri.shape
        if len(writes) != 2 or len(reads) != 2 or writes[0] != n or reads[0] != n or ww.shape != writes or (
                rw.shape != reads):
            raise ValueError('routes must be [sequences, selected banks]')
        if wi.dtype is not torch.int64 or ri.dtype is not torch.int64:
            raise ValueError('bank indices must be int64')
        if not (k.dtype is b.dtype is v.dtype is w.dtype is ww.dtype is rw.dtype is dtype):
            raise ValueError('controllers and route weights must share a dtype')
        if g.dtype is not torch.float32:
            g = g.float()
        index, pointers, copies = self._index, [], []
        for t in (q, k, b, v, w, ww, rw, g, wi, ri):
            if t.get_device() != index:
                raise ValueError('all tensors must be on the device of the pages')
            pointer = t.data_ptr()
            if pointer % 16 or not t.is_contiguous():
                t = t.clone(memory_format=torch.contiguous_format)
                copies.append(t)  # alive until the launch is enqueued
                pointer = t.data_ptr()
            pointers.append(pointer)
        kw, kr = writes[1], reads[1]
        output = torch.empty((n, heads * width), device=device, dtype=dtype)
        args = self._step
        (args.q, args.k, args.b, args.v, args.w, args.write_weights, args.read_weights, args.g, args.write_indices,
         args.read_indices) = pointers
        args.output, args.batch, args.write_banks, args.read_banks = output.data_ptr(), n, kw, kr
        args.ctrl_dtype, args.routed_decay, args.scale = ops._dtype_code(dtype), bool(routed_decay), scale
        self._call('bdm_pages_decode', layer, self._step_ref, self._tables.data_ptr(), self._tables.nbytes)
        return output
