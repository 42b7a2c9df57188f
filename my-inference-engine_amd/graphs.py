"""Captured decode steps: one HIP graph per batch bucket, replayed over static metadata buffers.

The reference launches every kernel of every decode step from Python (chat.py:257-308 drives
model.py:157-207 once per step); at 16 chats that launch overhead, not the GPU, sets the time per
output token.  This module captures the whole decode forward (28 layers: norms, projections,
fused RoPE + cache write, paged attention, MLP, final norm, logits) once per batch bucket
(1, 2, 4, 8, 16 rows by default) and replays it.  Sampling stays outside the graph.

What varies from step to step lives in device buffers the graph reads.  With the cache's
device-resident tables (the default on the GPU) that is only [row slots | token ids], one small
host-to-device copy per step: the graph itself starts with the metadata launch
(kernels.meta.step_metadata), which reads the rows' tables and lengths on the device, writes
starts, kv_lens, the batch block table and the new tokens' cache slots, and advances the lengths.
Without device tables the graph reads a host-packed [starts | kv_lens | block_table rows x W |
slot_mapping rows] buffer (KVCache.pack_step's layout) and the token ids, two copies per step.
Either way W = the most blocks one sequence may hold, so any sequence fits and the attention
kernel's grid and workspace (sized for W*block_size keys) never change: its work split follows the
actual kv_lens on the device.  A batch smaller than its bucket is padded with empty rows (slot -1: no keys,
nothing written to the cache, zeros from attention), whose logits are ignored.

Steps whose rows share enough of their blocks (KVCache.shared_groups, device tables only) replay
another graph of the bucket, whose attention reads them once; which rows share what comes up with the
slots and ids.  It is captured by capture_shared(), or when the first such step comes: two steps and a
capture in the middle of serving, and device memory for its intermediates (51 MB of workspace and more).  A
step for which that memory cannot be had replays the bucket's ordinary graph, which computes the same.
"""
import numpy as np
import torch

from kernels.meta import step_metadata
from kv_cache import SharedRows, StepMeta


def _out_of_memory(error):
    """Whether memory that could not be had is behind an error (ending a capture may raise another)."""
    while error is not None and not isinstance(error, torch.OutOfMemoryError):
        error = error.__context__
    return error is not None


class DecodeGraphs:
    def __init__(self, model, cache, buckets=(1, 2, 4, 8, 16)):
        assert cache.device.type == "cuda", "decode graphs need the GPU"
        self.model = model
        self.cache = cache
        self.W = cache.max_blocks_per_seq
        self.buckets = sorted(buckets)
        self.graphs = {}
        self.shared_graphs = {}     # by bucket, as they are needed
        self._no_shared = set()     # buckets whose sharing graph found no memory
        # One capture stream for all buckets, alive as long as the graphs: the kernels' workspace
        # is kept per stream, and a stream handle recycled by torch's pool while these graphs
        # exist would hand their workspace to unrelated calls.
        self._side = torch.cuda.Stream(device=cache.device)
        for rows in self.buckets:
            self._capture(rows)

    @property
    def max_rows(self):
        return self.buckets[-1]

    def _bucket(self, n):
        for b in self.buckets:
            if b >= n:
                return b
        raise ValueError(f"batch of {n} rows is larger than the largest captured bucket")

    def capture_shared(self, rows=None):
        """Capture the sharing graph of a bucket (default: of all that may replay one) now, so that no step
        has to.  Raises if there is no memory for it."""
        for bucket in self.buckets if rows is None else [self._bucket(rows)]:
            if self._may_share(bucket) and bucket not in self.shared_graphs:
                self._capture(bucket, shared=True)
                self._no_shared.discard(bucket)

    def _may_share(self, rows):
        return self.cache.device_tables and rows <= self.cache.SHARED_MAX_ROWS   # (padding rows count)

    def _shared_ready(self, rows):
        """Whether the bucket's sharing graph is there or can be captured."""
        if rows not in self.shared_graphs and rows not in self._no_shared:
            try:
                self.capture_shared(rows)
            except RuntimeError as error:
                if not _out_of_memory(error):
                    raise
                self._no_shared.add(rows)
        return rows in self.shared_graphs

    def _capture(self, rows, shared=False):
        dev, W, bs = self.cache.device, self.W, self.cache.block_size
        cache = self.cache
        if cache.device_tables:
            # [row slots | ids], and where rows share [cu_rows | prefix lengths]
            n_in = 4 * rows + 1 if shared else 2 * rows
            inp = torch.zeros(n_in, dtype=torch.int32, device=dev)
            inp[:rows] = -1                  # padding rows: nothing advances while warming up
            row_slots, ids_dev = inp[:rows], inp[rows:2 * rows].view(rows, 1)
            groups = None
            if shared:
                groups = SharedRows(rows=rows, cu_q=torch.arange(rows + 1, dtype=torch.int32,
                                                            device=dev),
                                    cu_rows=inp[2 * rows:3 * rows + 1],
                                    prefix_lens=inp[3 * rows + 1:], max_q=1)
            out = torch.zeros(2 * rows + rows * W + rows, dtype=torch.int32, device=dev)
            meta = StepMeta(starts=None, T=1, block_size=bs, starts_dev=out[:rows],
                            kv_lens=out[rows:2 * rows],
                            block_table=out[2 * rows:2 * rows + rows * W].view(rows, W),
                            slot_mapping=None, slot_mapping32=out[2 * rows + rows * W:],
                            kv_cap=W * bs, shared=groups)

            def step():
                step_metadata(cache, row_slots, None, 1, meta.starts_dev, meta.kv_lens,
                              meta.block_table, meta.slot_mapping32)
                return self.model.forward_meta(ids_dev, cache, meta)
            host = torch.zeros(n_in, dtype=torch.int32).pin_memory()
            # `out` is written by every replay: it lives as long as the graph (it was allocated
            # before the capture, so the graph's own memory pool does not hold it)
            bufs = (inp, host, out, groups)
        else:
            n_meta = 2 * rows + rows * W + rows
            meta_dev = torch.zeros(n_meta, dtype=torch.int32, device=dev)
            meta_dev[2 * rows + rows * W:] = -1      # no slot: nothing is written while warming up
            ids_dev = torch.zeros(rows, 1, dtype=torch.long, device=dev)
            meta = StepMeta(starts=None, T=1, block_size=bs, starts_dev=meta_dev[:rows],
                            kv_lens=meta_dev[rows:2 * rows],
                            block_table=meta_dev[2 * rows:2 * rows + rows * W].view(rows, W),
                            slot_mapping=None, slot_mapping32=meta_dev[2 * rows + rows * W:],
                            kv_cap=W * bs)

            def step():
                return self.model.forward_meta(ids_dev, cache, meta)
            bufs = (meta_dev, ids_dev, torch.zeros(n_meta, dtype=torch.int32).pin_memory(),
                    torch.zeros(rows, 1, dtype=torch.long).pin_memory())
        side = self._side
        side.wait_stream(torch.cuda.current_stream(dev))
        try:
            with torch.cuda.stream(side), torch.no_grad():
                for _ in range(2):                   # allocations and workspaces happen here
                    step()
        finally:      # a step that fails frees the buffers, which the work before it may still use
            torch.cuda.current_stream(dev).wait_stream(side)
        torch.cuda.synchronize(dev)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph), torch.no_grad():
            logits = step()
        kept = self.shared_graphs if shared else self.graphs
        kept[rows] = (graph, logits, bufs, torch.cuda.Event())

    def run(self, seqs, tokens):
        """One decode step for cache sequences `seqs` fed `tokens` (one id per row); returns the
        rows' logits [len(seqs), vocab] (a view of the graph's output buffer, valid until the next
        replay of the same bucket)."""
        n = len(seqs)
        rows = self._bucket(n)
        cache = self.cache
        groups = cache.shared_groups(seqs) if self._may_share(rows) else None
        if groups is not None and not self._shared_ready(rows):
            groups = None
        graph, logits, bufs, copied = (self.graphs if groups is None else self.shared_graphs)[rows]
        copied.synchronize()             # the previous upload from these host buffers is done
        if cache.device_tables:
            assert len(set(seqs)) == n, "a sequence may appear once per step"
            inp, host = bufs[:2]
            for s in seqs:
                cache.ensure_capacity(s, cache.length(s) + 1)
            h = host.numpy()
            h[:n] = [cache.slot[s] for s in seqs]
            h[n:rows] = -1
            h[rows:rows + n] = tokens
            h[rows + n:] = 0
            if groups is not None:
                cu, prefix = groups
                h[2 * rows:3 * rows + 1] = n                  # groups that are not there: empty
                h[2 * rows:2 * rows + len(cu)] = cu
                h[3 * rows + 1:3 * rows + 1 + len(prefix)] = prefix
            inp.copy_(host, non_blocking=True)
        else:
            meta_dev, ids_dev, host_meta, host_ids = bufs
            cache.pack_step(seqs, 1, W=self.W, out=host_meta.numpy(), rows=rows)
            ids = host_ids.numpy()
            ids[:n, 0] = tokens
            ids[n:, 0] = 0
            meta_dev.copy_(host_meta, non_blocking=True)
            ids_dev.copy_(host_ids, non_blocking=True)
        copied.record()
        graph.replay()
        cache.advance(seqs, 1)
        return logits[:n, -1]
