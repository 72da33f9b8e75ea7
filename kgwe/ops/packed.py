"""Packed batches: sequences of different lengths one after the other on one
token axis (``native/ops/packed_plan.hip``).

A ``PackedBatch`` holds what the kernels of such a batch need of its lengths:
where every sequence starts, each row's position, and the attention kernels'
job table (blocks of 128 rows, longest sweep first).  It is built on the GPU in
two small launches; make it once per batch and pass it to every layer.
"""
from __future__ import annotations

import torch

from ._lib import check, lib, ptr, raw_stream, stream

_INT32_MAX = 2**31 - 1


class PackedBatch:
    """Lengths of the sequences packed on one token axis of ``total`` rows.

    lengths: a list of ints (or a CPU integer tensor), or an integer tensor on
        the GPU.  Lengths of zero are allowed.
    total: rows of the token axis, by default the sum of the lengths; rows
        behind the last sequence are padding.  It has to be given where the
        lengths are on the GPU: they are not copied to the host, so they are
        not checked either; negative ones count as zero and what passes
        ``total`` is cut off.
    device: where the tables go; by default the lengths' device for a tensor
        on the GPU, else the current GPU, else the CPU.

    Attributes: ``n`` sequences, ``total``, ``device``, and int32 tensors
    ``cu`` [n + 2] (first row of every sequence, end of the last, total),
    ``positions`` [total] and ``seq_ids`` [total] (both -1 for padding rows),
    ``last_rows`` [n] (last row of every sequence; the row before it for an
    empty one).  The tables belong to the stream they were built on, like any
    tensor; built inside a graph capture (lengths on the GPU only) they belong
    to that graph, and a batch built before a capture that uses it has to be
    kept, like any input, as long as the graph is replayed.
    """

    def __init__(self, lengths, total: int | None = None, device=None):
        on_gpu = isinstance(lengths, torch.Tensor) and lengths.is_cuda
        if isinstance(lengths, torch.Tensor):
            if lengths.dim() != 1 or lengths.dtype not in (torch.int32, torch.int64):
                raise ValueError("PackedBatch: lengths must be int32 or int64 [n]")
        if on_gpu:
            if total is None:
                raise ValueError("PackedBatch: lengths on the GPU need total (they are not copied to the host)")
            device = lengths.device if device is None else torch.device(device)
            if device.type == "cuda" and device.index is None:
                device = torch.device("cuda", torch.cuda.current_device())
            if device != lengths.device:
                raise ValueError("PackedBatch: lengths on the GPU are planned on their own device")
            self.n = lengths.shape[0]
        else:
            values = [int(x) for x in (lengths.tolist() if isinstance(lengths, torch.Tensor) else lengths)]
            if any(x < 0 for x in values):
                raise ValueError("PackedBatch: lengths must not be negative")
            self.n = len(values)
            if total is None:
                total = sum(values)
            if sum(values) > total:
                raise ValueError(f"PackedBatch: the sequences have {sum(values)} rows, total is {total}")
            if device is None:
                device = "cuda" if torch.cuda.is_available() else "cpu"
            device = torch.device(device)
            if device.type == "cuda" and device.index is None:
                device = torch.device("cuda", torch.cuda.current_device())
        self.total = int(total)
        if not 0 <= self.total <= _INT32_MAX - 256:
            raise ValueError("PackedBatch: total must be in [0, 2^31 - 257]")
        if self.n > 1 << 24:
            raise ValueError("PackedBatch: at most 2^24 sequences")
        self.device = device
        if device.type != "cuda":
            self._plan_on_host(values)
            return
        with torch.cuda.device(device):
            if on_gpu:
                self.lengths = lengths.detach().clamp(0, self.total).to(torch.int32).contiguous()
            else:
                if torch.cuda.is_current_stream_capturing():  # the copy below would end the capture with an error
                    raise ValueError("PackedBatch: inside a graph capture lengths have to be on the GPU, with total")
                self.lengths = torch.tensor(values, dtype=torch.int32).to(device)
            self._plan_on_gpu()

    def _plan_on_host(self, values: list) -> None:
        i32 = {"dtype": torch.int32}
        starts, at = [], 0
        for x in values:
            starts.append(at)
            at += x
        self.lengths = torch.tensor(values, **i32)
        self.cu = torch.tensor([*starts, at, self.total], **i32)
        pad = torch.full((self.total - at,), -1, **i32)
        self.positions = torch.cat([*(torch.arange(x, **i32) for x in values), pad])
        self.seq_ids = torch.cat([*(torch.full((x,), i, **i32) for i, x in enumerate(values)), pad])
        self.jobs = None

    def _plan_on_gpu(self) -> None:
        n, T, dev = self.n, self.total, self.device
        self.cu = torch.zeros(n + 2, dtype=torch.int32, device=dev)
        self.positions = torch.empty(T, dtype=torch.int32, device=dev)
        self.seq_ids = torch.empty(T, dtype=torch.int32, device=dev)
        if T == 0:
            self.jobs = None
            return
        slots = int(lib().kgwe_packed_plan_jobs(n, T))
        self.jobs = torch.empty(slots, 4, dtype=torch.int32, device=dev)
        first = torch.empty(n + 2, dtype=torch.int32, device=dev)
        self._tables = (self.jobs.data_ptr(), slots)
        self._stream = raw_stream(dev.index)
        check(lib().kgwe_packed_plan(ptr(self.lengths), n, T, ptr(self.cu), ptr(first), ptr(self.jobs), slots,
                                     ptr(self.positions), ptr(self.seq_ids), stream(self.cu)), "packed_plan")

    @property
    def tables(self) -> tuple:
        """(job table, slots) for a launch on the current stream.  On another
        stream than the one they were built on, the table is marked as in use
        there: dropped while a kernel still reads it, its memory would be
        handed out again under that kernel."""
        if raw_stream(self.device.index) != self._stream:
            self.jobs.record_stream(torch.cuda.current_stream(self.device))
        return self._tables

    @property
    def last_rows(self) -> torch.Tensor:
        return self.cu[1:self.n + 1] - 1

    def __repr__(self) -> str:
        return f"PackedBatch(n={self.n}, total={self.total}, device={self.device})"
