"""Paged caches: host-side page bookkeeping around the HIP attention kernels.

Keeps the host protocol of the reference's cache object
(`tvm/llama_auto_batcher/llama_exec_graph.py:41-46,66,75-79,85,121-127`):
    add_sequence(sid) ; begin_forward(seq_ids, append_lens) ; attention_with_fused_qkv(layer, qkv, n_q_heads) ;
    end_forward()
with RoPE applied inside the cache operator (`llama_for_causal_lm.py:148-174`: rotary_dim = head_dim,
scale 1, no sliding window).  Keys are stored already rotated, which is equivalent to rotating them at
read time and saves the per-step re-rotation of the whole context.

A finished sequence gives its pages and its slot back with free_sequence(sid).  A sequence may begin with the whole pages of another
(share_prefix): they then have several owners and go back with the last of them.  Sequences may go on from all that another holds (fork), and
the beams of a search in one another's places (reorder).  Under a sliding window pages that no later token sees go back to the pool.

Device layout of PagedKVCache per layer: k [n_pages, Hkv, 16, D], v [n_pages, Hkv, D, 16] (fp16; in 8 bits that of ops.QuantPages), one int32 block table
[max_seqs, max_blocks], fp32 RoPE tables [max_pos, D/2].
"""
from __future__ import annotations

import numpy as np
import torch

from . import ops
from .decoder_ops import PrefillPlan, TimeMixPlan

PAGE = 16
AT_ONCE = 128       # sequences from which on a pass looks its pages up in one indexing


def rope_tables(head_dim: int, theta: float, max_pos: int):
    """cos/sin [max_pos, head_dim/2] float32 (float64 math, rounded once)."""
    inv_freq = theta ** (-(np.arange(0, head_dim, 2, dtype=np.float64) / head_dim))
    ang = np.arange(max_pos, dtype=np.float64)[:, None] * inv_freq[None, :]
    return np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)


class PageTable:
    """The host side of a paged cache: which pages of the pool belong to which sequence, and the protocol of a forward
    pass.  What lies in a page is up to the subclass."""

    shares_pages = True      # whether a page is all that its tokens leave behind
    plain = True             # whether the native passes and the plans over shared pages read it

    def __init__(self, n_pages, max_seqs, max_blocks, max_pos, device, free_pages=None, page_size=PAGE):
        if page_size != PAGE:
            raise ValueError(f"page_size must be {PAGE}")
        self.n_pages, self.max_seqs, self.max_blocks, self.max_pos = n_pages, max_seqs, max_blocks, max_pos
        self.device = torch.device(device)
        self.free = list(range(n_pages)) if free_pages is None else [int(p) for p in free_pages]
        if sorted(self.free) != list(range(n_pages)):
            raise ValueError("free_pages must be a permutation of range(n_pages)")
        # host mirrors (integer bookkeeping is host logic, as in the reference's runtime)
        self.table_h = np.full((max_seqs, max_blocks), -1, dtype=np.int32)
        self.lens = {}          # sid -> committed length
        self.slot = {}          # sid -> row of the block table
        self.free_slots = list(range(max_seqs))
        self._owners = {}       # page -> sequences, of the pages that have several
        self.block_table = torch.from_numpy(self.table_h.copy()).to(self.device)
        self._dirty = False
        self._cur = None
        self._staged = None     # (raw stream, event) of arrays queued last
        self._users = {}        # raw stream -> (stream, event behind the last pass's work or None): streams whose work reads the arrays
        self._adrift = {}       # sequences -> their slots [n] on the device, of beams whose rows the device has changed since the host read them

    # ------------------------------------------------------------------ protocol
    def add_sequence(self, sid):
        if sid in self.slot:
            raise ValueError(f"sequence with id {sid} has already been added")
        if not self.free_slots:
            raise RuntimeError("paged KV cache: no sequence slot left")
        self.slot[sid] = self.free_slots.pop(0)
        self.lens[sid] = 0

    def free_sequence(self, sid):
        """Give back the pages and the slot of a finished sequence."""
        if self._cur is not None:
            raise RuntimeError("free_sequence between begin_forward and end_forward")
        self.settle()
        row = self.slot.pop(sid)
        del self.lens[sid]
        for p in self.table_h[row][self.table_h[row] >= 0].tolist():
            self._own(p, -1)
        self.table_h[row] = -1
        self.free_slots.insert(0, row)
        self._dirty = True

    def _own(self, page, more):
        """`more` sequences take a page over, or give it back."""
        n = self._owners.get(page, 1) + more
        if n > 1:
            self._owners[page] = n
            return
        self._owners.pop(page, None)
        if n == 0:
            self.free.append(page)

    def settle(self):
        """Reads the rows of the block table back that a search's beams have on the device, where they have changed since: one wait for the device.  Pages
        that no beam holds any more go back to the pool.  Called by itself ahead of whatever needs the rows here."""
        if not self._adrift:
            return
        if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("paged KV cache: the rows of beams are to be read back, which a capture cannot")
        self._enter()
        table = self.block_table.cpu().numpy()
        for sids, slots in self._adrift.items():
            self._read_back(sids, slots.cpu().numpy(), table)
        self._adrift = {}

    def _read_back(self, sids, slots, table):
        rows = np.asarray([self.slot[s] for s in sids])
        if not np.array_equal(np.sort(rows), np.sort(slots)):
            raise RuntimeError(f"paged KV cache: beams of rows {rows.tolist()} in {slots.tolist()}")
        held = np.concatenate([self.table_h[rows].ravel(), table[rows].ravel()])
        pages, of = np.unique(held, return_inverse=True)
        n = held.size // 2
        for p, more in zip(pages.tolist(), (np.bincount(of.ravel()[n:], minlength=pages.size) - np.bincount(of.ravel()[:n], minlength=pages.size)).tolist()):
            if p >= 0 and more:
                self._own(p, more)
        self.table_h[rows] = table[rows]
        self.slot.update(zip(sids, slots.tolist()))

    def share_prefix(self, sid, of, tokens=None) -> int:
        """Sequence `sid`, added and still empty, begins with the first `tokens` tokens of sequence `of` (None: all that are committed),
        as far as they fill whole pages; returns how many that are.  The caller answers for the tokens being the same, and for
        whatever else makes their keys and values (the adapter)."""
        if self._cur is not None:
            raise RuntimeError("share_prefix between begin_forward and end_forward")
        if not self.shares_pages:
            raise ValueError(f"{type(self).__name__}: what a sequence leaves behind lies not in pages alone")
        self.settle()
        row, src = self.slot[sid], self.slot[of]
        if sid == of or self.lens[sid] or (self.table_h[row] >= 0).any():
            raise ValueError(f"share_prefix: sequence {sid} is not another, empty one")
        n = max(min(self.lens[of] if tokens is None else int(tokens), self.lens[of]), 0) // PAGE
        n = self._shareable(src, n)
        for p in self.table_h[src, :n].tolist():
            if p >= 0:
                self._own(p, 1)
        self.table_h[row, :n] = self.table_h[src, :n]
        self.lens[sid] = n * PAGE
        self._dirty = self._dirty or n > 0
        return n * PAGE

    def _shareable(self, row, n):
        """How many of a row's first n pages another sequence can begin with."""
        return n

    def _held(self, sid):
        """Blocks of a sequence that have had their pages."""
        return int((self.table_h[self.slot[sid]] >= 0).sum())

    def _release(self, seq_ids):
        """Ahead of a pass of these sequences, whatever of theirs it does not read."""

    def lacks_page(self, sid):
        """Whether the sequence's next token needs a page that it has not."""
        j = self.lens[sid] // PAGE
        return j < self.max_blocks and self.table_h[self.slot[sid], j] < 0

    def reserve(self, seq_ids, tokens):
        """Pages for the next `tokens` tokens of sequences, as far as their rows go and if the pool has all of them; otherwise none."""
        self.settle()
        room = min(self.max_blocks, self.max_pos // PAGE)
        want = [(self.slot[s], j) for s in seq_ids for j in range(self._held(s), min(-(-(self.lens[s] + tokens) // PAGE), room))]
        if want and len(want) <= len(self.free):
            for row, j in want:
                self.table_h[row, j] = self.free.pop(0)
            self._dirty = True

    def prefix_groups(self, seq_ids):
        """(positions in seq_ids, pages): which of the sequences begin with the same pages, cut so that the pages saved are most; of equal
        cuts one with fewer groups.

        The sequences' whole pages make a tree, whose nodes are what several of them begin with.  A group is a node, and every sequence
        goes with the deepest one that it passes: saved are the depths of the sequences' groups, less every group's own.  So from the leaves up,
        for each ancestor that may be the deepest group above a node: the most that its sequences save, with a group of their own at the node
        or without."""
        if any(s in sids for sids in self._adrift for s in seq_ids):
            self.settle()
        rows = [self.slot[s] for s in seq_ids]
        full = [self.lens[s] // PAGE for s in seq_ids]
        owned = [i for i, r in enumerate(rows) if full[i] and int(self.table_h[r, 0]) in self._owners]
        if len(owned) < 2:
            return []
        paths = {i: self.table_h[rows[i], :full[i]] for i in owned}
        # the tree from the sequences in the order of their pages, where neighbours share most
        depth, up, ends, below = [0], [0], [[]], [[]]         # of a node: its pages, parent, sequences that end there, children (node 0: no page)

        def node(d, parent):
            depth.append(d), up.append(parent), ends.append([]), below.append([])
            below[parent].append(len(depth) - 1)
            return len(depth) - 1

        last, at = None, 0
        for i in sorted(owned, key=lambda i: paths[i].tobytes()):
            n = 0
            if last is not None:
                n = min(full[last], full[i])
                differ = np.flatnonzero(paths[last][:n] != paths[i][:n])
                n = int(differ[0]) if differ.size else n
            under = None
            while depth[at] > n:
                under, at = at, up[at]
            if depth[at] < n:                                  # what the two share ends between two nodes
                mid = node(n, at)
                below[at].remove(under)
                below[mid].append(under)
                up[under], at = mid, mid
            if full[i] > n:
                at = node(full[i], at)
            ends[at].append(i)
            last = i
        order = [0]                                            # parents ahead of their children
        for v in order:
            order.extend(below[v])
        above = {0: np.zeros(1, np.int64)}                     # depths of the ancestors that may be the group above (node 0: none)
        for v in order:
            if below[v]:
                above.update(dict.fromkeys(below[v], above[0] if v == 0 else np.append(above[v], depth[v])))
        without, own, best = {}, {}, {}
        for v in reversed(order[1:]):
            without[v] = len(ends[v]) * above[v] + sum(best[c][:-1] for c in below[v])
            own[v] = (len(ends[v]) - 1) * depth[v] + sum(int(best[c][-1]) for c in below[v])
            best[v] = np.maximum(without[v], own[v])
        groups, group, which = [], {0: None}, {0: 0}           # of a node: the group that its sequences go with, its place among the ancestors
        for v in order[1:]:
            group[v], which[v] = group[up[v]], which[up[v]]
            if own[v] > without[v][which[v]]:
                group[v], which[v] = ([], depth[v]), len(above[v])
                groups.append(group[v])
            if group[v] is not None:
                group[v][0].extend(ends[v])
        return sorted((sorted(members), pages) for members, pages in groups)

    def begin_forward(self, seq_ids, append_lens, device_meta=None):
        """Reserve pages for the appended tokens and stage the per-token (sequence, position) arrays."""
        if self._cur is not None:
            raise RuntimeError("begin_forward called twice without end_forward")
        if len(seq_ids) != len(append_lens):
            raise ValueError("seq_ids and append_lens differ in length")
        self._release(seq_ids)
        if self._adrift and (device_meta is None or self._dirty):      # (a table that changes is uploaded whole, the beams' rows with it)
            self.settle()
            self._release(seq_ids)
        # Which sequences lack a page (they are handed out in order: the last one needed is missing).  us a step without host-made arrays, one by one / all at
        # once: one sequence 2.5 / 15.5, four 3.6 / 16.3, 64 29 / 34, 212 94 / 81
        if len(seq_ids) < AT_ONCE:
            short = []
            for sid, n in zip(seq_ids, append_lens):
                row, new_len = self.slot[sid], self.lens[sid] + n
                need = -(-new_len // PAGE)
                if new_len > self.max_pos or need > self.max_blocks:
                    raise RuntimeError(f"sequence {sid}: length {new_len} exceeds the cache geometry")
                if need > 0 and self.table_h[row, need - 1] < 0:
                    short.append((sid, need))
        else:
            rows, base = self._rows_and_lens(seq_ids)
            new_len = base + np.asarray(append_lens, dtype=np.int64)
            need = -(-new_len // PAGE)
            beyond = (new_len > self.max_pos) | (need > self.max_blocks)
            if beyond.any():
                i = int(beyond.argmax())
                raise RuntimeError(f"sequence {seq_ids[i]}: length {new_len[i]} exceeds the cache geometry")
            short = [(seq_ids[i], int(need[i])) for i in np.flatnonzero((need > 0) & (self.table_h[rows, np.maximum(need, 1) - 1] < 0))]
        if short and self._adrift:
            self.settle()
            return self.begin_forward(seq_ids, append_lens, device_meta)
        for sid, need in short:
            row = self.slot[sid]
            for j in range(self._held(sid), need):
                if not self.free:
                    raise RuntimeError("paged KV cache out of pages")
                self.table_h[row, j] = self.free.pop(0)
                self._dirty = True
        self._enter()
        staged = self._dirty or device_meta is None
        if self._dirty:
            self.block_table.copy_(ops.upload(torch.from_numpy(self.table_h), self.device))
            self._dirty = False
        decode = all(n == 1 for n in append_lens)
        if device_meta is not None:
            tok_seq, tok_pos, ctx = device_meta
        elif decode:
            rows, base = self._rows_and_lens(seq_ids)
            tok_seq, tok_pos, ctx = ops.upload(torch.from_numpy(np.stack([rows, base, base + 1])), self.device)
        else:
            rows, base = self._rows_and_lens(seq_ids)
            ts = np.repeat(rows, append_lens).astype(np.int32)
            tp = np.concatenate([b + np.arange(n, dtype=np.int32) for b, n in zip(base, append_lens)]).astype(np.int32)
            tok_seq, tok_pos = ops.upload(torch.from_numpy(np.stack([ts, tp])), self.device)
            ctx = None
        if staged:
            self._stage()
        self._cur = (list(seq_ids), list(append_lens), decode, tok_seq, tok_pos, ctx)

    def _rows_and_lens(self, seq_ids):
        """Block-table rows and lengths of sequences."""
        return np.asarray([self.slot[s] for s in seq_ids], dtype=np.int32), np.asarray([self.lens[s] for s in seq_ids], dtype=np.int32)

    # Host-made arrays are queued on the stream that is current, not waited for, and the next pass overwrites the block table.  So a
    # stream that goes on with a pass waits for its arrays, and the stream that begins the next one waits for all that the last was
    # queued on.  No event from outside may enter a capture: one begins behind a wait for the whole device, or on a stream that its
    # caller has ordered.
    def _raw_stream(self):
        return torch._C._cuda_getCurrentRawStream(self.block_table.device.index)

    def _enter(self):
        """A pass begins on the current stream."""
        if self.device.type != "cuda" or torch.cuda.is_current_stream_capturing():
            return
        raw = self._raw_stream()
        stream = self._users[raw][0] if raw in self._users else torch.cuda.current_stream(self.device)
        for r, (other, behind) in self._users.items():
            if r != raw:
                stream.wait_stream(other) if behind is None else stream.wait_event(behind)
        self._users = {raw: (stream, None)}

    def _stage(self):
        """Arrays of the pass have been queued on the current stream."""
        if self.device.type == "cuda" and not torch.cuda.is_current_stream_capturing():
            raw = self._raw_stream()
            if raw not in self._users:
                self._users[raw] = (torch.cuda.current_stream(self.device), None)
            self._staged = (raw, self._users[raw][0].record_event())

    def _join(self):
        """The pass goes on on the current stream."""
        if self.device.type != "cuda":
            return
        raw = self._raw_stream()
        elsewhere = self._staged is not None and raw != self._staged[0]
        if (raw in self._users and not elsewhere) or torch.cuda.is_current_stream_capturing():
            return
        stream = torch.cuda.current_stream(self.device)
        self._users[raw] = (stream, None)
        if elsewhere:
            stream.wait_event(self._staged[1])
            for t in self._pass_arrays():          # their memory may be given out again, to the stream they were made on
                t.record_stream(stream)

    def __getstate__(self):
        """A copy, or a pickle, is made behind all that the passes have queued and knows no streams (which neither takes)."""
        self.settle()
        self._enter()
        return {**self.__dict__, "_staged": None, "_users": {}}

    def _pass_arrays(self):
        """Arrays that were made for the current pass."""
        return [t for t in self._cur[3:] if t is not None]

    def end_forward(self):
        seq_ids, append_lens = self._cur[0], self._cur[1]
        for sid, n in zip(seq_ids, append_lens):
            self.lens[sid] += n
        self.abandon_forward()

    def abandon_forward(self):
        """Ends a pass that failed: its sequences are as long as before.  (What it may have stored behind their ends is written anew; the tokens of an 8-bit
        cache's last page outlast a step, not a pass that went on to another page.)"""
        self._cur = None
        for raw, (stream, _) in self._users.items():         # (the default stream outlives every pass: no event before one is waited for)
            if raw and not torch.cuda.is_current_stream_capturing():
                self._users[raw] = (stream, stream.record_event())

    # ------------------------------------------------------------------ helpers
    def rows_of(self, seq_ids):
        """The rows of the block table that sequences have."""
        self.settle()
        return [self.slot[s] for s in seq_ids]

    def pages_of(self, sid):
        self.settle()
        row = self.table_h[self.slot[sid]]
        return row[row >= 0].tolist()


class PagedKVCache(PageTable):
    def __init__(self, n_layers, n_pages, n_kv_heads, head_dim, max_seqs, max_blocks, rope_theta, max_pos,
                 device="cuda:0", free_pages=None, page_size=PAGE, n_q_heads=None, bits=16, window=None, sinks=0):
        """n_q_heads: of the model that reads the cache; without them decode steps read shared pages for each sequence anew.
        bits: 8 holds every page that is complete in 8 bits, at a step per page and head (ops.QuantPages), in little more than half the memory.
        window: a token sees only the last so many, itself among them, and the first `sinks`; pages in between go back to the pool.  Positions stay those of the text.
        A cache of either kind is read by operators of its own, one launch a layer and step (`plain` is false)."""
        super().__init__(n_pages, max_seqs, max_blocks, max_pos, device, free_pages, page_size)
        if bits not in (8, 16):
            raise ValueError(f"PagedKVCache: pages of {bits} bits (8 or 16)")
        self.bits, (self.window, self.sinks) = bits, ops._window("PagedKVCache", window, sinks)
        self.plain = bits == 16 and not self.window
        if not self.plain and head_dim not in (64, 128):
            raise ValueError(f"PagedKVCache: pages of {bits} bits with a window of {window} tokens for heads of {head_dim} (64 or 128)")
        self.cut = None         # tokens by which attention over a cache that is not plain shares its work out
        self._gone = {}         # sid -> block in front of which all but the sinks' have gone back
        self.n_layers, self.Hkv, self.D, self.n_q_heads = n_layers, n_kv_heads, head_dim, n_q_heads
        self.plan = None        # of the current decode step
        self._plans = {}        # batch -> SharedPrefixPlan or None, for batches whose sequences are there
        if head_dim % 32:
            raise ValueError("head_dim must be a multiple of 32")
        # keys in matrix-core fragment order: element (token, d) of a page at [d // 32, (d % 32) // 8, token, d % 8]
        zeros = lambda *shape, dtype=torch.float16: torch.zeros((n_layers, *shape), dtype=dtype, device=self.device)      # noqa: E731
        last = (max_seqs if bits == 8 else n_pages, n_kv_heads)
        k16, v16 = zeros(*last, head_dim // 32, 4, PAGE, 8), zeros(*last, head_dim, PAGE)
        if bits == 8:
            self.tail_k, self.tail_v, self._pages = k16, v16, {}
            self.k = zeros(n_pages, n_kv_heads, head_dim // 64, 4, PAGE, 2, 8, dtype=torch.int8)
            self.v = zeros(n_pages, n_kv_heads, head_dim // 64, 4, PAGE, 4, 4, dtype=torch.int8)
            self.step = zeros(n_pages, n_kv_heads, 2, dtype=torch.float32)
        else:
            self.k, self.v = k16, v16
        cos, sin = rope_tables(head_dim, rope_theta, max_pos)
        self.rope_cos = torch.from_numpy(cos).to(self.device)
        self.rope_sin = torch.from_numpy(sin).to(self.device)

    def k_rowmajor(self, layer: int) -> torch.Tensor:
        """The layer's rotated keys as [n_pages, Hkv, 16, D] (a copy, for inspection; of pages in 8 bits what they stand for)."""
        if self.bits == 8:
            return self.pages(layer).values(torch.arange(self.n_pages, dtype=torch.int32, device=self.device))[0]
        k = self.k[layer]
        return k.permute(0, 1, 4, 2, 3, 5).reshape(self.n_pages, self.Hkv, PAGE, self.D).contiguous()

    def pages(self, layer) -> ops.QuantPages:
        """A layer's pages in 8 bits."""
        if layer not in self._pages:
            self._pages[layer] = ops.QuantPages(self.k[layer], self.v[layer], self.step[layer], self.tail_k[layer], self.tail_v[layer])
        return self._pages[layer]

    def __getstate__(self):
        state = super().__getstate__()
        return {**state, "_pages": {}} if self.bits == 8 else state

    # Under a window a row has the pages of the sinks, then none, then those from the first one on that its next token sees.
    def _first_seen(self, length):
        return max(length - self.window + 1, 0) // PAGE if self.window else 0

    def _release(self, seq_ids):
        if not self.window:
            return
        adrift = {s for sids in self._adrift for s in sids}      # (rows that are not known here keep their pages until they are)
        for sid in seq_ids:
            first, gone = self._first_seen(self.lens[sid]), self._gone.get(sid, -(-self.sinks // PAGE))
            if first > gone and sid not in adrift:
                blocks = self.table_h[self.slot[sid], gone:first]
                for p in blocks[blocks >= 0].tolist():
                    self._own(p, -1)
                blocks[:] = -1
                self._gone[sid] = first
                self._dirty = True

    def _held(self, sid):
        if not self.window:
            return super()._held(sid)
        has = np.flatnonzero(self.table_h[self.slot[sid]] >= 0)
        return max(int(has[-1]) + 1 if has.size else 0, -(-self.lens[sid] // PAGE))

    def _shareable(self, row, n):
        if not self.window:
            return n
        seen = np.arange(n)
        seen = seen[(seen < -(-self.sinks // PAGE)) | (seen >= self._first_seen(n * PAGE))]
        return n if (self.table_h[row, seen] >= 0).all() else 0  # (a row that has gone on may have given back what this one needs)

    def fork(self, sids, of):
        """Sequences `sids`, which are added here, go on from all the tokens of sequence `of`: its whole pages have them as owners too, the contents of its
        last page are copied (all sequences and layers in one launch)."""
        if self._cur is not None:
            raise RuntimeError("fork between begin_forward and end_forward")
        sids = list(sids)
        self.settle()
        src, n = self.slot[of], self.lens[of]
        full, part = n // PAGE, n % PAGE > 0
        if len(set(sids)) < len(sids) or any(s in self.slot for s in sids):
            raise ValueError("fork: a sequence that has already been added")
        if len(sids) > len(self.free_slots) or part and len(sids) > len(self.free):
            raise RuntimeError(f"paged KV cache: {len(self.free_slots)} slots and {len(self.free)} pages left for {len(sids)} sequences")
        pairs = []
        for sid in sids:
            self.add_sequence(sid)
            row = self.slot[sid]
            for p in self.table_h[src, :full].tolist():
                if p >= 0:
                    self._own(p, 1)
            self.table_h[row, :full] = self.table_h[src, :full]
            if part:
                self.table_h[row, full] = self.free.pop(0)
                pairs.append((src, row) if self.bits == 8 else (int(self.table_h[src, full]), int(self.table_h[row, full])))
            self.lens[sid] = n
            if of in self._gone:
                self._gone[sid] = self._gone[of]
        self._dirty = self._dirty or bool(sids)
        if pairs:
            try:
                self._enter()
                at = ops.upload(torch.tensor(pairs, dtype=torch.int32).t().contiguous(), self.device)
                ops.copy_pages([self.tail_k, self.tail_v] if self.bits == 8 else [self.k, self.v], at[0], at[1])
            except Exception:
                for sid in sids:
                    self.free_sequence(sid)
                raise

    def reorder(self, sids, parents, slots, ctx):
        """A step of a beam search: the beams `sids` of requests (an equal number each, one behind the other, of equal length) go on from the tokens of their parents [R, W]
        int32 (-1: from none), chosen by ops.beam_select.  slots [R * W] int32 are their rows of the block table, and become those that they then have; ctx [R * W] their lengths.
        All of it stays on the device, can be recorded into a graph, and is one launch for the rows and one for what is to be copied: the contents of last pages
        that are not complete.  The host learns of it from `adrift`."""
        new, moves = ops.beam_reorder(parents, slots, self.block_table, ctx)
        if self.bits == 8:
            ops.copy_pages([self.tail_k, self.tail_v], moves.src_slot, moves.dst_slot)
        else:
            ops.copy_pages([self.k, self.v], moves.src_page, moves.dst_page)
        slots.copy_(new)

    def adrift(self, sids, slots):
        """`reorder` of these beams has run, or is queued (or will be, behind the pass that has begun): their rows are to be read back (`settle`) before they are used here."""
        sids = tuple(sids)
        self._adrift[sids] = slots
        if self.plain:
            # the batch's own plan, if it has one by now, is of the pages that its requests' beams shared first, and share on: none is made of others
            self._plans.setdefault(sids, None)
            if len(self._plans) > 1:
                self._plans = {b: p for b, p in self._plans.items() if b == sids or not set(b) & set(sids)}

    def free_sequence(self, sid):
        super().free_sequence(sid)
        self._gone.pop(sid, None)
        self._plans = {b: p for b, p in self._plans.items() if sid not in b}

    def share_prefix(self, sid, of, tokens=None):
        n = super().share_prefix(sid, of, tokens)
        self._plans = {b: p for b, p in self._plans.items() if sid not in b}
        return n

    def shared_plan(self, seq_ids):
        """The plan by which a decode step of these sequences reads the pages they share once, or None where none are shared or it does
        not pay.  Kept while all of them live (recorded steps read it), and cut anew where their own pages have outgrown it (looked at when the
        first of them has filled a page).  A pass that is being recorded takes the plan that is there, or none.  us of attention without / with, 50 own tokens a row:
        32 heads of 128 over 32, 32 rows, 16 shared pages 16.4 / 14.2, 64 pages 35 / 16, 256 pages 133 / 29; 2 rows, 64 pages 11.2 / 10.4, 256 pages
        38 / 22; 128 rows, 4 pages 36 / 35; 32 heads over 8, 32 rows, 64 pages (130 MB) 12.8 / 14.6, 256 pages 32 / 23, 128 rows, 16 pages (133 MB) 18 / 16,
        64 rows, 64 pages 20 / 17."""
        if not self._owners or not self.plain or not self.n_q_heads or not 1 <= self.n_q_heads // self.Hkv <= 16:
            return None
        batch = tuple(seq_ids)
        recorded = self.device.type == "cuda" and torch.cuda.is_current_stream_capturing()      # (a capture takes no arrays from the host)
        if batch not in self._plans:
            if recorded:
                return None
            groups = self.prefix_groups(batch)
            saved = sum((len(m) - 1) * p for m, p in groups) * self.Hkv * self.D * 4 * PAGE
            pays = saved >= 132e6 or any(p >= 128 for _, p in groups)
            self._plans[batch] = self._cut(batch, groups, saved) if pays else None
        plan = self._plans[batch]
        if plan is not None and not recorded and self.lens[batch[0]] % PAGE == 0 and plan.outgrown([self.lens[s] + 1 for s in batch]):
            self._plans[batch] = self._cut(batch, plan.groups, plan.saved_bytes)
            self._plans[batch].earlier = plan
        return self._plans[batch]

    def _cut(self, batch, groups, saved):
        plan = ops.SharedPrefixPlan(groups, [self.lens[s] + 1 for s in batch], self.n_q_heads, self.Hkv, self.D, self.device)
        plan.saved_bytes = saved
        self._stage()
        return plan

    def begin_forward(self, seq_ids, append_lens, device_meta=None):
        super().begin_forward(seq_ids, append_lens, device_meta)
        if not self.plain:
            # a step's work is cut for the next power of two, so that a recorded one is cut as the others are
            longest = max((self.lens[s] + n for s, n in zip(seq_ids, append_lens)), default=0)
            self.cut = min(max(1 << max(longest - 1, 0).bit_length(), 256), self.max_blocks * PAGE) if self._cur[2] else longest
        self.plan = self.shared_plan(seq_ids) if self._cur[2] and self._owners else None
        if self.plan is not None and self.device.type == "cuda" and not torch.cuda.is_current_stream_capturing():
            self.plan.data.record_stream(torch.cuda.current_stream(self.device))      # (it may have been made on another)

    def _pass_arrays(self):
        return super()._pass_arrays() + ([self.plan.data] if self.plan is not None else [])

    def attention_with_fused_qkv(self, layer, qkv, n_q_heads, out=None, frag=False, o_shrink=None):
        """qkv [T, Hq + 2 Hkv, D] (or [T, (Hq + 2 Hkv) * D]) fp16, token-major in begin_forward order.
        Rotates q in place, appends rotated k and v, attends causally; returns [T, Hq * D] fp16
        (frag=True: as a FragActivation ready for the o_proj product).  o_shrink (a decode step only): see
        ops.paged_attn_decode - the call then returns (attention output, head shares of the o projection's shrink)."""
        if self._cur is None:
            raise RuntimeError("attention_with_fused_qkv outside begin_forward/end_forward")
        self._join()
        _, append_lens, decode, tok_seq, tok_pos, ctx = self._cur
        T = sum(append_lens)
        qkv = qkv.view(T, n_q_heads + 2 * self.Hkv, self.D)
        if not self.plain:
            if o_shrink is not None:
                raise ValueError("attention_with_fused_qkv: o_shrink is for plain caches")
            return self._attention(layer, qkv, n_q_heads, out, frag)
        ops.rope_kv_append(qkv, self.k[layer], self.v[layer], self.block_table, tok_seq, tok_pos,
                           self.rope_cos, self.rope_sin, n_q_heads, self.Hkv, self.D)
        if decode and self.plan is not None and n_q_heads == self.n_q_heads and o_shrink is None:
            return ops.paged_attn_decode_shared(qkv, self.k[layer], self.v[layer], self.block_table, tok_seq, ctx, self.plan, n_q_heads, self.Hkv, self.D,
                                                out=out, frag=frag)
        if decode:
            return ops.paged_attn_decode(qkv, self.k[layer], self.v[layer], self.block_table, tok_seq, ctx,
                                         n_q_heads, self.Hkv, self.D, out=out, frag=frag, o_shrink=o_shrink)
        if o_shrink is not None:
            raise ValueError("attention_with_fused_qkv: o_shrink is for decode steps")
        return ops.paged_attn_prefill(qkv, self.k[layer], self.v[layer], self.block_table, tok_seq, tok_pos,
                                      n_q_heads, self.Hkv, self.D, out=out, frag=frag)

    def _attention(self, layer, qkv, n_q_heads, out, frag):
        """`attention_with_fused_qkv` of a cache in 8 bits, or under a window (which may leave q as it comes)."""
        _, _, decode, tok_seq, tok_pos, _ = self._cur
        where, heads = (self.block_table, tok_seq, tok_pos), (n_q_heads, self.Hkv, self.D)
        seen = {"window": self.window or None, "sinks": self.sinks, "longest": self.cut, "out": out, "frag": frag}
        rope = (self.rope_cos, self.rope_sin)
        if self.bits == 8:
            return (ops.rope_attn_decode_q8 if decode else ops.rope_attn_prefill_q8)(qkv, self.pages(layer), *where, *rope, *heads, **seen)
        k, v = self.k[layer], self.v[layer]
        if decode:
            return ops.rope_attn_decode_window(qkv, k, v, *where, *rope, *heads, **seen)
        ops.rope_kv_append(qkv, k, v, *where, *rope, *heads)
        return ops.paged_attn_prefill_window(qkv, k, v, *where, *heads, **seen)

    def kv_bytes_read_per_step(self, seq_ids):
        """Algorithmic K+V bytes one decode step reads for these sequences, all layers."""
        per_pos = self.n_layers * 2 * self.Hkv * self.D * 2
        seen = [n if not self.window or n <= self.window + self.sinks else self.window + self.sinks for n in (self.lens[s] + 1 for s in seq_ids)]
        if self.bits == 8:                       # complete pages at a byte a number and two steps, those ahead of the token's own
            own = [(self.lens[s] % PAGE) + 1 for s in seq_ids]
            return int(sum(o * per_pos + (n - o) * (per_pos // 2 + self.n_layers * self.Hkv * 8 // PAGE) for n, o in zip(seen, (min(o, n) for o, n in zip(own, seen)))))
        return int(sum(seen)) * per_pos


class PagedLatentCache(PageTable):
    """Pages of latent attention: per layer one vector per token, the normed latent and the rotated key part, in the page
    layout of latent_attention.hip.  A layer may read another layer's pages instead of having its own."""

    def __init__(self, layers, n_pages, max_seqs, max_blocks, max_pos, dtype, device="cuda:0", free_pages=None, page_size=PAGE):
        """layers: per layer (kv_rank, rot_dim, rotation, owner): owner is the layer whose pages this one reads (itself,
        if it has its own); rotation: rotary.Rotation."""
        super().__init__(n_pages, max_seqs, max_blocks, max_pos, device, free_pages, page_size)
        self.dtype = dtype
        self.owner = [o for *_, o in layers]
        self.pages = []
        self.rope = []
        tables = {}
        for l, (rank, rot_dim, rotation, o) in enumerate(layers):
            blocks = -(-rank // 32) + -(-rot_dim // 32)
            # padding between and behind the two parts is read by the matrix cores: it stays zero
            self.pages.append(torch.zeros((n_pages, blocks, 4, PAGE, 8), dtype=dtype, device=self.device) if o == l else self.pages[o])
            key = (rotation, rot_dim)
            if key not in tables:
                tables[key] = tuple(torch.from_numpy(t).to(self.device) for t in rotation.tables(rot_dim, max_pos))
            self.rope.append(tables[key])
        self._plan = None

    def latents(self, layer, sid):
        """The cached vectors [length, blocks * 32] of a sequence (a copy, for inspection)."""
        n = self.lens[sid]
        p = self.pages[layer][torch.tensor(self.pages_of(sid), device=self.device, dtype=torch.int64)]
        return p.permute(0, 3, 1, 2, 4).reshape(-1, p.shape[1] * 32)[:n].contiguous()

    def latent_attention(self, layer, qkv, att, out=None):
        """The mixer of `layer` behind its input projection: qkv [T, att.proj_rows] in begin_forward order (att:
        latent_attention.LatentAttention) -> the heads' outputs, concatenated (`out`: an activation of att.out_cols
        columns)."""
        if self._cur is None:
            raise RuntimeError("latent_attention outside begin_forward/end_forward")
        self._join()
        seq_ids, append_lens, _, tok_seq, tok_pos, _ = self._cur
        ctx = [self.lens[s] + n for s, n in zip(seq_ids, append_lens)]
        return att.attend(qkv, self.pages[layer], self.block_table, tok_seq, tok_pos, *self.rope[layer], max_ctx=max(ctx),
                          store=self.owner[layer] == layer, plan=self.attention_plan(att), out=out)

    def _pass_arrays(self):
        plan = self._plan[1] if self._plan is not None and self._plan[0] is self._cur else None
        return super()._pass_arrays() + ([plan.tiles, plan.phys] if plan is not None else [])

    def attention_plan(self, att):
        """The pass's plan for the prompt form where `att` takes that (one serves all layers), else None."""
        seq_ids, append_lens, decode = self._cur[:3]
        if decode:
            return None
        ctx = [self.lens[s] + n for s, n in zip(seq_ids, append_lens)]
        if not att.prompt_form_pays(list(zip(append_lens, ctx))):
            return None
        if self._plan is None or self._plan[0] is not self._cur:
            self._plan = (self._cur, PrefillPlan([(self.pages_of(s), n, c) for s, n, c in zip(seq_ids, append_lens, ctx)], self.device, wait=False))
            self._stage()
        return self._plan[1]


class PagedStateCache(PageTable):
    """What the layers of a model with recurrent and attention layers keep per sequence, one entry per layer run (a layer that
    runs several times has one for every pass): pages of tied attention, or a state per slot.  A slot needs no clearing:
    kernels start a sequence's state from zero at its position 0."""

    shares_pages = False

    def __init__(self, runs, width_p, n_pages, max_seqs, max_blocks, max_pos, dtype, device="cuda:0", free_pages=None, page_size=PAGE):
        """runs: per layer run the mixer's spec, whose cache_entry says what is kept; width_p: columns of the residual stream."""
        super().__init__(n_pages, max_seqs, max_blocks, max_pos, device, free_pages, page_size)
        self.dtype = dtype
        self.entries = [tuple(torch.zeros(shape, dtype=dtype if elements else torch.float32, device=self.device)
                              for shape, elements in s.cache_entry(n_pages, max_seqs, PAGE, width_p)) for s in runs]
        self._meta = None

    def values(self, run, sid):
        """The cached values [length, G, columns] of a sequence (a copy, for inspection)."""
        p = self.entries[run][0][torch.tensor(self.pages_of(sid), device=self.device, dtype=torch.int64)]
        return p.permute(0, 4, 1, 2, 3, 5).reshape(-1, p.shape[1], p.shape[2] * 32)[: self.lens[sid]].contiguous()

    def state(self, run, sid):
        """The matrix states [H, D, D] of a sequence (a view)."""
        return self.entries[run][0][self.slot[sid]]

    def shift(self, run):
        """The previous tokens' rows [slots, columns] of a recurrent layer run."""
        return self.entries[run][1]

    def _pass(self):
        """Of the current pass, made once for all its layers: {"last": the last token of every token's sequence, "segs": [n][4]
        {slot, first token, tokens, position}} - both None in a decode step - and the plans of the prompt forms, once taken."""
        if self._cur is None:
            raise RuntimeError("outside begin_forward/end_forward")
        self._join()
        if self._meta is None or self._meta[0] is not self._cur:
            seq_ids, lens, decode = self._cur[:3]
            m = {"last": None, "segs": None, "plan": None, "ranges": {}, "host": None}
            if not decode:
                ends = np.cumsum(lens)
                m["host"] = segs = [(self.slot[s], int(e) - n, n, self.lens[s]) for s, n, e in zip(seq_ids, lens, ends)]
                both = np.concatenate([np.asarray(segs, dtype=np.int32).reshape(-1), np.repeat(ends - 1, lens).astype(np.int32)])
                both = ops.upload(torch.from_numpy(both), self.device)
                self._stage()
                m["segs"], m["last"] = both[: 4 * len(segs)].view(-1, 4), both[4 * len(segs):]
            self._meta = (self._cur, m)
        return self._meta[1]

    def _pass_arrays(self):
        out, m = super()._pass_arrays(), self._meta[1] if self._meta is not None and self._meta[0] is self._cur else {}
        if m.get("segs") is not None:
            out += [m["segs"], m["last"]]
        if m.get("plan") is not None:
            out += [m["plan"].tiles, m["plan"].phys]
        return out + [a for r in m.get("ranges", {}).values() for a in (r.ranges, r.seqs)]

    def token_meta(self):
        """(sequence, position, last token of its sequence in the pass) per token."""
        return self._cur[3], self._cur[4], self._pass()["last"]

    def time_mix(self, run, mixes, mixer):
        """The recurrence of a layer run on the five mixes of the pass (mixer: time_mix.TimeMix)."""
        m = self._pass()
        return mixer.run(mixes, self.entries[run][0], m["segs"], self._cur[3], self._cur[4], self.time_mix_plan(mixer))

    def time_mix_plan(self, mixer):
        """The pass's ranges where `mixer` takes the prompt form, else None."""
        m, heads = self._pass(), mixer.spec.heads
        if m["host"] is None or not mixer.prompt_form:
            return None
        if heads not in m["ranges"]:
            m["ranges"][heads] = TimeMixPlan(m["host"], heads, self.device, wait=False)
            self._stage()
        return m["ranges"][heads]

    def attention_plan(self, att):
        """The pass's plan where `att` takes the prompt form, else None."""
        m = self._pass()
        seq_ids, append_lens, decode = self._cur[:3]
        seqs = [(n, self.lens[s] + n) for s, n in zip(seq_ids, append_lens)]
        if decode or not att.prompt_form_pays(seqs):
            return None
        if m["plan"] is None:
            m["plan"] = PrefillPlan([(self.pages_of(s), n, c) for s, (n, c) in zip(seq_ids, seqs)], self.device, wait=False)
            self._stage()
        return m["plan"]

    def tied_attention(self, run, y, att):
        """The attention of a layer run behind its input projection y (att: tied_attention.TiedAttention)."""
        if self._cur is None:
            raise RuntimeError("outside begin_forward/end_forward")
        seq_ids, append_lens, _, tok_seq, tok_pos, _ = self._cur
        max_ctx = max(self.lens[s] + n for s, n in zip(seq_ids, append_lens))
        return att.attend(y, *self.entries[run], self.block_table, tok_seq, tok_pos, max_ctx=max_ctx, plan=self.attention_plan(att))
