"""Paged KV cache feeding the MI355X paged attention kernels.

Same layout and bookkeeping as the reference's KVCache (kv_cache.py:8-121): one buffer
[num_layers, 2, num_blocks * block_size, num_kv_heads, head_dim] (dim 1: k=0, v=1), a free list of
blocks, per-sequence block tables, and logical token p of a sequence at physical slot
table[p // block_size] * block_size + p % block_size (kv_cache.py:15-16).  The API (alloc, free,
length, blocks_needed, ensure_capacity, trim, prepare, advance, write, read) keeps the reference's
names and meaning.

What changes is the per-step metadata.  The reference builds a Python list per new token and a
dense [B, S] gather index every step (kv_cache.py:74-101), then copies every cached token of every
row into a dense tensor per layer (kv_cache.py:117-121).  Here prepare() builds, with vectorised
numpy and ONE pinned host-to-device copy, exactly what the paged kernel reads:

  * block_table [B, W] int32 (rows padded with block 0, kv_cache.py:95),
  * kv_lens [B] int32 (keys per row after this step, model.py:175),
  * slot_mapping [B*T] (where this step's new tokens go, for write()),

and no per-layer gather happens on the GPU path.  read() (the dense gather) is kept for the CPU
fallback and for reference-compatible callers.

On the GPU the tables themselves are device-resident (device_tables, the default there): every
sequence holds a slot with a row of `dev_tables` [max_seqs, max_blocks_per_seq] int32 and a
length in `dev_lens` [max_seqs] int32 (both bounded independently of the pool size, so the tables
stay small for a pool of any size: 4096 x 2048 x 4 B = 32 MB at most by default).  A table row is written only when blocks are allocated
(ensure_capacity: one small copy per allocation), and a step sends only its rows' slots: one HIP
launch (kernels.meta.step_metadata, csrc/step_meta.hip) derives starts, kv_lens, the batch block
table, every new token's slot (and positions / last indices for mixed steps) and advances the
device lengths in place.  The host keeps the same tables and lengths for scheduling decisions.

prepare_packed() builds the metadata of a mixed step, where each row appends its own number of
tokens (one for a decoding chat, a whole prompt for a newly admitted one) and the rows' tokens are
packed back to back: prefix offsets cu_q, every token's position and slot, and each row's last
token (whose logits are sampled).

Beyond the reference, blocks can have several holders: fork() makes sequences over another's history
that share its whole blocks (a count per block says when it is free again), copy_from() brings a
sequence over from another cache and compact() moves the blocks in use together.  A step whose rows
share enough carries which rows share what (SharedRows), and its attention reads the shared blocks
once (kernels.shared).
"""
import math
import operator
from collections import Counter
from dataclasses import dataclass, field

import numpy as np
import torch


@dataclass
class SharedRows:
    """Which of a step's first `rows` rows hold the same first blocks: kernels.shared's arguments."""
    rows: int
    cu_q: torch.Tensor           # [rows+1] int32: prefix offsets of their new tokens
    cu_rows: torch.Tensor        # [G+1] int32: rows [cu_rows[g], cu_rows[g+1]) share
    prefix_lens: torch.Tensor    # [G] int32: this many tokens
    max_q: int                   # new tokens of a row, at most


@dataclass
class StepMeta:
    """Metadata of one forward step over rows `seqs`, each appending T tokens."""
    starts: list                 # tokens each row held before this step (host ints)
    T: int
    block_size: int
    starts_dev: torch.Tensor     # [B] int32
    kv_lens: torch.Tensor        # [B] int32 = starts + T
    slot_mapping: torch.Tensor   # [B*T] int64, row-major (row, t)
    block_table: torch.Tensor    # [B, W] int32
    slot_mapping32: torch.Tensor = None  # the same slots as int32 (for the fused RoPE + write)
    tables: list = field(default_factory=list)  # host copies of the rows' block lists
    kv_cap: int = None           # fixed upper bound of kv_lens (captured decode graphs)
    shared: SharedRows = None    # None: no rows that share enough
    packed = False

    @property
    def max_kv(self):
        return self.kv_cap if self.kv_cap is not None else max(self.starts) + self.T

    def gather_idx(self, device):
        """[B, S] physical slot of every logical position [0, max_kv) (kv_cache.py:93-98)."""
        S, bs = self.max_kv, self.block_size
        pos = torch.arange(S, device=device)
        bt = self.block_table.to(device).long()
        return bt[:, pos // bs] * bs + pos % bs


@dataclass
class PackedMeta:
    """Metadata of one mixed step: row b appends counts[b] >= 1 tokens, packed back to back in row
    order (row b's tokens are [cu_q[b], cu_q[b+1]) of the packed batch)."""
    starts: list                 # tokens each row held before this step (host ints)
    counts: list                 # new tokens per row (host ints)
    block_size: int
    n_single: int                # leading rows with exactly one new token (decode-shaped rows)
    cu_q: torch.Tensor           # [B+1] int32
    kv_lens: torch.Tensor        # [B] int32 = starts + counts
    positions: torch.Tensor      # [N] int32: position of each packed token in its row
    slot_mapping32: torch.Tensor  # [N] int32: cache slot of each packed token
    last_idx: torch.Tensor       # [B] int32: packed index of each row's last token
    block_table: torch.Tensor    # [B, W] int32
    tables: list = field(default_factory=list)
    shared: SharedRows = None    # None: no rows that share enough
    packed = True

    def split(self, D=None):
        """(max kv_len of the leading D rows (default: the one-token rows), of the other rows, max
        new tokens of the other rows): the host bounds each attention launch is sized by."""
        D = self.n_single if D is None else D
        kv = [s + c for s, c in zip(self.starts, self.counts)]
        return (max(kv[:D], default=0), max(kv[D:], default=0), max(self.counts[D:], default=0))

    @property
    def max_kv(self):
        return max(s + c for s, c in zip(self.starts, self.counts))

    @property
    def max_q(self):
        return max(self.counts)

    @property
    def slot_mapping(self):
        return self.slot_mapping32.long()


def _common(a, b):
    """Leading blocks that two tables have in common: they share those of a fork and none after, so the
    last one is found by halving."""
    lo, hi = 0, min(len(a), len(b))
    if not hi or a[0] != b[0]:
        return 0
    while lo < hi:
        mid = (lo + hi + 1) // 2
        if a[mid - 1] == b[mid - 1]:
            lo = mid
        else:
            hi = mid - 1
    return lo


class KVCache:
    # Default cap of one sequence's length: Qwen2.5's context window.
    DEFAULT_MAX_TOKENS_PER_SEQ = 32768
    DEFAULT_MAX_SEQS = 4096
    # K and V bytes that a step would read again in a layer, from which its attention reads the shared
    # blocks once (sharing_pays has what else counts).  With less to save the plain kernels' smaller
    # fixed cost wins.  us of a layer's attention shared / plain, K and V not in the caches, one new token:
    # 16 rows over 1,024 shared keys of 2 heads (16 MB) 15.2 / 13.7, over 2,048 (31 MB) 15.5 / 17.0; 4 rows over 4,096
    # of 4 (25 MB) 14.6 / 17.4, of 8 (50 MB) 16.6 / 22.5; 64 rows over 31,000 of 2 (2.0 GB) 38 / 251.
    SHARED_BYTES = 20 << 20
    # New tokens of a row up to which it may pay: with more its own tiles are full, and sharing saves no
    # matrix products.
    SHARED_MAX_NEW = 32
    SHARED_MAX_ROWS = 512     # rows of a call of the kernel

    def __init__(self, num_blocks, block_size, device, dtype, num_layers, num_kv_heads, head_dim,
                 *, device_tables=None, max_seqs=None, max_blocks_per_seq=None):
        self.buf = torch.zeros(num_layers, 2, num_blocks * block_size, num_kv_heads, head_dim,
                               device=device, dtype=dtype)
        self.num_blocks = num_blocks
        self.block_size = block_size
        self.device = torch.device(device)
        self._free_blocks = list(range(num_blocks))
        self._block_tables = {}   # seq id -> list of block ids, in logical order
        self._lengths = {}        # seq id -> tokens written so far
        self._next_seq = 0
        self._holders = [0] * num_blocks   # sequences that hold each block
        self._extra = 0                    # holders beyond a block's first, over all blocks
        # The tree of forks, for order(): a sequence's parent and its forks.  A freed sequence stays while
        # at least two of its branches live, so there are fewer of those than sequences.
        self._above, self._below = {}, {}
        self.device_tables = self.device.type == "cuda" if device_tables is None else device_tables
        # Blocks one sequence may hold.  With device tables this is the width of a table row: the
        # pool, capped at the default context length, so the tables do not grow with the square
        # of the pool.  Host tables limit nothing, so there (as in the reference's KVCache) a
        # sequence may hold the whole pool unless the caller sets a cap.
        if max_blocks_per_seq is None:
            max_blocks_per_seq = (math.ceil(self.DEFAULT_MAX_TOKENS_PER_SEQ / block_size)
                                  if self.device_tables else num_blocks)
        self.max_blocks_per_seq = max(1, min(num_blocks, max_blocks_per_seq))
        # Sequence slots (rows of the device tables).  Every sequence that holds cache holds at
        # least one block once its first token is written, so num_blocks + a few transient empty
        # sequences bound how many can be live; the default takes that bound up to 4096 slots (the
        # scheduler evicts idle conversations when slots run out).
        if max_seqs is None:
            max_seqs = min(num_blocks + 16, self.DEFAULT_MAX_SEQS)
        self.max_seqs = max_seqs
        self._free_slots = list(range(self.max_seqs - 1, -1, -1))
        self.slot = {}            # seq id -> slot
        if self.device_tables:
            assert self.device.type == "cuda", "device-resident tables need a GPU cache"
            self.dev_tables = torch.zeros(self.max_seqs, self.max_blocks_per_seq, dtype=torch.int32,
                                          device=device)
            self.dev_lens = torch.zeros(self.max_seqs, dtype=torch.int32, device=device)

    # -- bookkeeping (kv_cache.py:31-72) -------------------------------------------------------
    def free_block_count(self):
        return len(self._free_blocks)

    def free_slot_count(self):
        return len(self._free_slots)

    def blocks_needed(self, seq, total_len):
        held = len(self._block_tables[seq]) if seq is not None else 0
        return max(0, math.ceil(total_len / self.block_size) - held)

    def alloc(self):
        seq = self._new_seq()
        if self.device_tables:
            slot = self.slot[seq]
            self.dev_lens[slot:slot + 1].zero_()
        return seq

    def _new_seq(self, parent=None):
        if not self._free_slots:
            raise RuntimeError(f"all {self.max_seqs} sequence slots are in use")
        seq = self._next_seq
        self._next_seq += 1
        self._block_tables[seq] = []
        self._lengths[seq] = 0
        self.slot[seq] = self._free_slots.pop()
        self._above[seq], self._below[seq] = parent, set()
        if parent is not None:
            self._below[parent].add(seq)
        return seq

    def free(self, seq):
        self._release(self._block_tables.pop(seq))
        del self._lengths[seq]
        self._free_slots.append(self.slot.pop(seq))
        self._prune(seq)

    def _prune(self, node):
        """Take a freed sequence that joins no two branches out of the tree of forks."""
        while node is not None and node not in self._lengths and len(self._below[node]) < 2:
            above, below = self._above.pop(node), self._below.pop(node)
            if above is not None:
                self._below[above].remove(node)
                self._below[above] |= below
            for child in below:
                self._above[child] = above
            node = above       # it may have joined this branch and one more

    def _take(self, n):
        """n free blocks, now held once each."""
        blocks = [self._free_blocks.pop() for _ in range(n)]
        for b in blocks:
            self._holders[b] = 1
        return blocks

    def _release(self, blocks):
        """One holder fewer for each; free again are those without."""
        for b in blocks:
            self._holders[b] -= 1
            if self._holders[b] == 0:
                self._free_blocks.append(b)
            else:
                self._extra -= 1

    def length(self, seq):
        return self._lengths[seq]

    def ensure_capacity(self, seq, total_len):
        need = self.blocks_needed(seq, total_len)
        if need > len(self._free_blocks):
            raise RuntimeError(f"KV cache exhausted: seq {seq} needs {need} more blocks, "
                               f"only {len(self._free_blocks)} free")
        if len(self._block_tables[seq]) + need > self.max_blocks_per_seq:
            raise RuntimeError(f"seq {seq} would hold {len(self._block_tables[seq]) + need} blocks; "
                               f"a sequence holds at most {self.max_blocks_per_seq}")
        table = self._block_tables[seq]
        old = len(table)
        table.extend(self._take(need))
        if self.device_tables and need:
            new = torch.tensor(table[old:], dtype=torch.int32)
            self.dev_tables[self.slot[seq], old:old + need].copy_(new)

    def trim(self, seq):
        table = self._block_tables[seq]
        keep = math.ceil(self._lengths[seq] / self.block_size)
        self._release(table[keep:])
        del table[keep:]

    # -- blocks with several holders (no counterpart in the reference) ----------------------------
    def fork(self, seq, n=1, length=None):
        """n new sequences that begin with the first `length` tokens of seq (default: all it holds).

        They share its whole blocks and get a copy of the one that is only started, so that each
        writes its next tokens into a block of its own: one launch over all layers.  Returns their
        ids.  Raises before anything changes if blocks or sequence slots are short."""
        length = self._lengths[seq] if length is None else operator.index(length)
        if not 0 <= length <= self._lengths[seq]:
            raise ValueError(f"seq {seq} holds {self._lengths[seq]} tokens, not {length}")
        n, bs, table = operator.index(n), self.block_size, self._block_tables[seq]
        whole, rest = divmod(length, bs)
        need = n if rest else 0
        if n < 1:
            raise ValueError(f"{n} forks")
        if need > len(self._free_blocks):
            raise RuntimeError(f"KV cache exhausted: {n} forks of seq {seq} need {need} blocks, "
                               f"only {len(self._free_blocks)} free")
        if n > len(self._free_slots):
            raise RuntimeError(f"{n} forks of seq {seq}: only {len(self._free_slots)} of "
                               f"{self.max_seqs} sequence slots are free")
        fresh = self._take(need)
        forks = []
        for i in range(n):
            child = self._new_seq(seq)
            self._block_tables[child] = table[:whole] + fresh[i:i + 1]
            self._lengths[child] = length
            forks.append(child)
        for b in table[:whole]:
            self._holders[b] += n
        self._extra += n * whole
        try:
            if self.device_tables:
                from kernels.blocks import fork_rows
                slot = self.slot[seq]
                rows = [[slot, self.slot[c], length, fresh[i] if rest else -1]
                        for i, c in enumerate(forks)]
                fork_rows(self.buf, self.dev_tables, self.dev_lens, self._upload(rows).view(n, 4), bs)
            elif rest:
                self._copy([(table[whole], b) for b in fresh])
        except Exception:
            for child in forks:
                self.free(child)
            raise
        return forks

    def copy_from(self, other, seq):
        """A new sequence holding what `seq` of another cache (of the same layers, heads, dtype,
        block size and device) holds; returns its id."""
        if self.buf.shape[:2] != other.buf.shape[:2] or self.buf.shape[3:] != other.buf.shape[3:] or (
                self.buf.dtype, self.buf.device, self.block_size) != (
                other.buf.dtype, other.buf.device, other.block_size):
            raise ValueError("copy_from needs caches of one layout, dtype, block size and device")
        length = other._lengths[seq]
        mine = self.alloc()
        try:
            self.ensure_capacity(mine, length)
            self._copy(list(zip(other._block_tables[seq], self._block_tables[mine])), other)
            if self.device_tables:
                slot = self.slot[mine]
                self.dev_lens[slot:slot + 1].fill_(length)
        except Exception:
            self.free(mine)
            raise
        self._lengths[mine] = length
        return mine

    def compact(self):
        """Move the blocks in use to the lowest ids, 0 .. n - 1, and return n: buf[:, :, :n *
        block_size] then holds every sequence.  One launch; the next blocks handed out follow them."""
        used = sum(h > 0 for h in self._holders)
        src = [b for b in range(used, self.num_blocks) if self._holders[b]]
        dst = [b for b in range(used) if not self._holders[b]]
        new_ids = list(range(self.num_blocks))
        pairs = list(zip(src, dst))
        for a, b in pairs:
            new_ids[a] = b
        if pairs and self.device_tables:
            from kernels.blocks import move_blocks
            rows = [(self.slot[s], len(t)) for s, t in self._block_tables.items() if t]
            ids = self._upload(pairs + rows, new_ids)
            n, m = 2 * len(pairs), 2 * (len(pairs) + len(rows))
            move_blocks(self.buf, self.dev_tables, ids[n:m].view(-1, 2), ids[:n].view(-1, 2), ids[m:],
                        self.block_size)
        else:
            self._copy(pairs)
        # (the books follow what was moved)
        for a, b in pairs:
            self._holders[b], self._holders[a] = self._holders[a], 0
        if pairs:
            for table in self._block_tables.values():
                table[:] = [new_ids[b] for b in table]
        self._free_blocks = list(range(self.num_blocks - 1, used - 1, -1))
        return used

    def reclaimable(self, seqs):
        """Blocks that freeing all of `seqs` would give back: those that no other sequence holds."""
        held = Counter(b for s in seqs for b in self._block_tables[s])
        return sum(self._holders[b] == n for b, n in held.items())

    def order(self, seqs):
        """Indices that put sequences which share blocks next to each other: forks after what they
        were forked from.  Sequences that share nothing keep their order."""
        if not self._extra:
            return list(range(len(seqs)))
        paths = {None: ()}     # from the root of its tree to a sequence
        first, keys = {}, []   # where each tree begins; a row's place
        for i, s in enumerate(seqs):
            todo, at = [], s
            while at not in paths:
                todo.append(at)
                at = self._above[at]
            path = paths[at]
            for at in reversed(todo):
                path = paths[at] = path + (at,)
            keys.append((first.setdefault(path[0], i), path))
        return sorted(range(len(seqs)), key=keys.__getitem__)

    def shared_groups(self, seqs):
        """(cu_rows, prefix tokens) of neighbouring rows that hold the same first blocks, or None if a
        step of one token a row would gain too little by reading them once."""
        groups = self._groups(seqs)
        return groups if groups is not None and self.sharing_pays(seqs, groups) else None

    def _groups(self, seqs):
        if not self._extra or not 2 <= len(seqs) <= self.SHARED_MAX_ROWS:
            return None
        cu, prefix = [0], []
        rows, blocks = 1, 0       # of the group being formed
        tables = [self._block_tables[s] for s in seqs]
        for a, b in zip(tables, tables[1:]):
            same = _common(a, b)
            joined = min(same, blocks) if rows > 1 else same
            # one more row, at the price of a shorter prefix for all
            if joined and rows * joined >= (rows - 1) * blocks:
                rows, blocks = rows + 1, joined
                continue
            cu.append(cu[-1] + rows)
            prefix.append(blocks * self.block_size)
            rows, blocks = 1, 0
        cu.append(cu[-1] + rows)
        prefix.append(blocks * self.block_size)
        return cu, prefix

    def sharing_pays(self, seqs, groups, new_tokens=None, splits=False, walk=0):
        """Whether a step over `seqs` gains by reading what `groups` (cu_rows, prefix tokens) share once:
        whether the bytes it would read again outweigh what the shared kernel costs more.  That grows with

          the bytes that remain: it reads them at 5.4 TB/s, the plain decode kernel at 5.9
          the rows: each has two parts to merge.  64 rows over 512 shared keys of 2 heads (33 MB saved)
            take 17.6 us, plain 16.1; 256 rows of 500 keys, four of which share 16,384 more, 61.5 / 52.4
          new_tokens (of all rows, default one each) beyond one a row: more pairs of each, 16 rows of up
            to 16 over 512 keys of 8 heads 26.0 / 20.6
          the tokens of a row where the plain kernel would cut its keys into pieces (splits: a step of
            equal rows, few enough for it): 8 rows of 8 over 8,192 keys of 2 heads 25.9 / 22.5

        and falls with the keys that a row of several tokens has (walk) where it does not cut them: there
        one work-group walks them all (the same 8,192 keys under 32 rows 37.0 / 210.2), which the shared
        kernel deals out.  All in proportion to SHARED_BYTES.  Of 1,373 measured steps with up to 32 new
        tokens a row the rule sends 918 to the kernel, four of which are slower there by more than 5 %."""
        cu, prefix = groups
        rows = len(seqs)
        more = 0 if new_tokens is None else new_tokens - rows
        token = 2 * self.buf.shape[3] * self.buf.shape[4] * self.buf.element_size()
        saved = sum((b - a - 1) * p for a, b, p in zip(cu, cu[1:], prefix))
        rest = sum(self._lengths[s] for s in seqs) + rows + more - saved
        cost = 1 + rest * token / (480 << 20) + rows / 52 + more / 110
        if splits:
            cost += 0.75 * more / rows
        else:
            cost = max(cost - walk / 700, 0.3)   # (0.3: none that saves less was measured)
        return saved * token >= self.SHARED_BYTES * cost

    def _shared_rows(self, seqs, counts, cu_q=None, query_heads=None):
        """The SharedRows of a step over `seqs`, or None; cu_q if they are on the device already (a packed
        step)."""
        if not self._extra or self.device.type != "cuda":
            return None
        rows = 0      # the leading ones with few new tokens
        while rows < len(seqs) and counts[rows] <= self.SHARED_MAX_NEW:
            rows += 1
        seqs, counts = seqs[:rows], counts[:rows]
        if max(counts, default=1) == 1:
            groups = self.shared_groups(seqs)
        else:
            groups = self._groups(seqs)
            # fa2_paged cuts the keys of a step of equal rows that leave compute units without work
            splits = cu_q is None and (query_heads or 1) * rows <= 256
            walk = max(self._lengths[s] + c for s, c in zip(seqs, counts) if c > 1)
            if groups is not None and not self.sharing_pays(seqs, groups, sum(counts), splits, walk):
                groups = None
        if groups is None:
            return None
        cu, prefix = groups
        g = len(prefix)
        offsets = [] if cu_q is not None else np.concatenate([[0], np.cumsum(counts)])
        up = self._upload(cu, prefix, offsets)
        return SharedRows(rows=rows, cu_q=up[2 * g + 1:] if cu_q is None else cu_q[:rows + 1],
                          cu_rows=up[:g + 1], prefix_lens=up[g + 1:2 * g + 1], max_q=max(counts))

    def _upload(self, *parts):
        """Lists of numbers (or of rows of them) as one flat int32 tensor on the device."""
        host = np.concatenate([np.asarray(p, dtype=np.int32).reshape(-1) for p in parts])
        return torch.from_numpy(host).pin_memory().to(self.device, non_blocking=True)

    def _copy(self, pairs, source=None):
        """Whole blocks, (from, to), in every layer; from another cache's buffer if given."""
        src = (source or self).buf
        if not pairs:
            return
        if self.device.type == "cuda":
            from kernels.blocks import copy_blocks
            copy_blocks(src, self.buf, self._upload(pairs).view(-1, 2), self.block_size)
            return
        at = torch.arange(self.block_size)
        a, b = ((torch.tensor(ids)[:, None] * self.block_size + at).reshape(-1) for ids in zip(*pairs))
        self.buf[:, :, b] = src[:, :, a]

    def advance(self, seqs, T):
        """Count T new tokens (an int, or one count per row) as written."""
        counts = T if isinstance(T, (list, tuple)) else [T] * len(seqs)
        for s, c in zip(seqs, counts):
            self._lengths[s] += c

    # -- per-step metadata ----------------------------------------------------------------------
    def pack_step(self, seqs, T, W=None, out=None, rows=None):
        """Grow the rows' tables for T new tokens and pack the step's metadata into one int32 host
        array [starts | kv_lens | block_table rows*W | slot_mapping rows*T] (kv_cache.py:74-101).

        W defaults to the blocks the longest row needs; `rows` >= len(seqs) pads the batch with
        empty rows (no keys, slot -1: nothing read or written).  Returns (array, starts, W)."""
        bs = self.block_size
        starts = [self._lengths[s] for s in seqs]
        for s, start in zip(seqs, starts):
            self.ensure_capacity(s, start + T)
        B = len(seqs)
        R = rows or B
        W = W or max(1, math.ceil((max(starts) + T) / bs))
        tables = [self._block_tables[s] for s in seqs]
        n_all = 2 * R + R * W + R * T
        host = np.zeros(n_all, dtype=np.int32) if out is None else out[:n_all]
        if out is not None:
            host.fill(0)
        st = np.asarray(starts, dtype=np.int32)
        host[:B] = st
        host[R:R + B] = st + T
        bt = host[2 * R:2 * R + R * W].reshape(R, W)
        for i, t in enumerate(tables):
            n = min(len(t), W)
            bt[i, :n] = t[:n]
        pos = st[:, None] + np.arange(T, dtype=np.int32)[None, :]        # [B, T]
        sm = host[2 * R + R * W:].reshape(R, T)
        sm[:B] = bt[np.arange(B)[:, None], pos // bs] * bs + pos % bs
        sm[B:] = -1
        return host, starts, W

    def prepare(self, seqs, T, query_heads=None):
        """The metadata of a step that appends T tokens to each of seqs.  query_heads: the model's, which
        decide with T > 1 from how much on shared blocks are read once (unknown: from more)."""
        if self.device_tables:
            return self._prepare_device(seqs, [T] * len(seqs), packed=False, query_heads=query_heads)
        B = len(seqs)
        host, starts, W = self.pack_step(seqs, T)
        tables = [self._block_tables[s] for s in seqs]
        cpu = torch.from_numpy(host)
        if self.device.type == "cuda":
            dev = cpu.pin_memory().to(self.device, non_blocking=True)
        else:
            dev = cpu.clone()
        return StepMeta(
            starts=starts, T=T, block_size=self.block_size,
            starts_dev=dev[:B], kv_lens=dev[B:2 * B],
            block_table=dev[2 * B:2 * B + B * W].view(B, W),
            slot_mapping=dev[2 * B + B * W:].long(),
            slot_mapping32=dev[2 * B + B * W:],
            tables=[list(t) for t in tables], shared=self._shared_rows(seqs, [T] * B, None, query_heads))

    def prepare_packed(self, seqs, counts):
        """Grow the rows' tables for counts[b] new tokens each and build a PackedMeta with one
        pinned host-to-device copy of [cu_q | kv_lens | positions | slots | last_idx | tables]."""
        assert len(seqs) == len(counts) and len(seqs) > 0 and min(counts) >= 1
        if self.device_tables:
            return self._prepare_device(seqs, counts, packed=True)
        bs = self.block_size
        starts = [self._lengths[s] for s in seqs]
        for s, start, c in zip(seqs, starts, counts):
            self.ensure_capacity(s, start + c)
        B, N = len(seqs), sum(counts)
        st = np.asarray(starts, dtype=np.int32)
        cnt = np.asarray(counts, dtype=np.int32)
        kv = st + cnt
        W = max(1, math.ceil(int(kv.max()) / bs))
        tables = [self._block_tables[s] for s in seqs]
        host = np.zeros(2 * B + 1 + 2 * N + B + B * W, dtype=np.int32)
        cu = host[:B + 1]
        np.cumsum(cnt, out=cu[1:])
        host[B + 1:2 * B + 1] = kv
        o = 2 * B + 1
        row = np.repeat(np.arange(B), cnt)                          # row of each packed token
        pos = host[o:o + N]
        pos[:] = st[row] + (np.arange(N, dtype=np.int32) - cu[:-1][row])
        bt = host[o + 2 * N + B:].reshape(B, W)
        for i, t in enumerate(tables):
            n = min(len(t), W)
            bt[i, :n] = t[:n]
        host[o + N:o + 2 * N] = bt[row, pos // bs] * bs + pos % bs
        host[o + 2 * N:o + 2 * N + B] = cu[1:] - 1
        n_single = 0
        while n_single < B and counts[n_single] == 1:
            n_single += 1
        cpu = torch.from_numpy(host)
        if self.device.type == "cuda":
            dev = cpu.pin_memory().to(self.device, non_blocking=True)
        else:
            dev = cpu.clone()
        return PackedMeta(
            starts=starts, counts=list(counts), block_size=bs, n_single=n_single,
            cu_q=dev[:B + 1], kv_lens=dev[B + 1:2 * B + 1], positions=dev[o:o + N],
            slot_mapping32=dev[o + N:o + 2 * N], last_idx=dev[o + 2 * N:o + 2 * N + B],
            block_table=dev[o + 2 * N + B:].view(B, W), tables=[list(t) for t in tables],
            shared=self._shared_rows(seqs, counts, dev[:B + 1]))

    def _prepare_device(self, seqs, counts, packed, query_heads=None):
        """The device-table path of prepare / prepare_packed: one pinned copy of the rows' slots
        (and packed offsets), one metadata launch; tables and lengths never leave the device."""
        from kernels.meta import step_metadata
        assert len(set(seqs)) == len(seqs), "a sequence may appear once per step"
        bs = self.block_size
        starts = [self._lengths[s] for s in seqs]
        for s, start, c in zip(seqs, starts, counts):
            self.ensure_capacity(s, start + c)
        B, N = len(seqs), sum(counts)
        W = max(1, math.ceil(max(st + c for st, c in zip(starts, counts)) / bs))
        host = np.empty(B + (B + 1 if packed else 0), dtype=np.int32)
        host[:B] = [self.slot[s] for s in seqs]
        if packed:
            host[B] = 0
            np.cumsum(np.asarray(counts, dtype=np.int32), out=host[B + 1:])
        small = torch.from_numpy(host).pin_memory().to(self.device, non_blocking=True)
        row_slots, cu = small[:B], (small[B:] if packed else None)
        out = torch.empty(3 * B + B * W + 2 * N, dtype=torch.int32, device=self.device)
        o_starts, o_kv, o_last = out[:B], out[B:2 * B], out[2 * B:3 * B]
        o_bt = out[3 * B:3 * B + B * W].view(B, W)
        o_slots, o_pos = out[3 * B + B * W:3 * B + B * W + N], out[3 * B + B * W + N:]
        step_metadata(self, row_slots, cu, counts[0], o_starts, o_kv, o_bt, o_slots,
                      o_pos if packed else None, o_last if packed else None)
        tables = [list(self._block_tables[s]) for s in seqs]
        if not packed:
            return StepMeta(starts=starts, T=counts[0], block_size=bs, starts_dev=o_starts,
                            kv_lens=o_kv, slot_mapping=None, block_table=o_bt,
                            slot_mapping32=o_slots, tables=tables,
                            shared=self._shared_rows(seqs, counts, None, query_heads))
        n_single = 0
        while n_single < B and counts[n_single] == 1:
            n_single += 1
        return PackedMeta(starts=starts, counts=list(counts), block_size=bs, n_single=n_single,
                          cu_q=cu, kv_lens=o_kv, positions=o_pos, slot_mapping32=o_slots,
                          last_idx=o_last, block_table=o_bt, tables=tables,
                          shared=self._shared_rows(seqs, counts, cu))

    # -- data movement --------------------------------------------------------------------------
    def k_pool(self, layer):
        return self.buf[layer, 0]

    def v_pool(self, layer):
        return self.buf[layer, 1]

    def write(self, layer, meta, k, v):
        """Scatter this step's k/v [B, Hkv, T, d] into their slots (kv_cache.py:108-115)."""
        B, H, T, D = k.shape
        sm = meta.slot_mapping if meta.slot_mapping is not None else meta.slot_mapping32.long()
        self.buf[layer, 0].index_copy_(0, sm, k.transpose(1, 2).reshape(B * T, H, D))
        self.buf[layer, 1].index_copy_(0, sm, v.transpose(1, 2).reshape(B * T, H, D))

    def read_row(self, layer, table, n):
        """Dense [Hkv, n, d] copies of the first n keys/values of the sequence whose block list is
        `table`: one row of read()."""
        pos = torch.arange(n, device=self.buf.device)
        idx = torch.tensor(table, device=self.buf.device, dtype=torch.long)[pos // self.block_size]
        idx = idx * self.block_size + pos % self.block_size
        return self.buf[layer, 0][idx].transpose(0, 1), self.buf[layer, 1][idx].transpose(0, 1)

    def read(self, layer, meta):
        """Dense [B, Hkv, S, d] copies of every row's keys/values (kv_cache.py:117-121)."""
        idx = meta.gather_idx(self.buf.device)
        return (self.buf[layer, 0][idx].transpose(1, 2), self.buf[layer, 1][idx].transpose(1, 2))
