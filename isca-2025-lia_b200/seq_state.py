"""Per-sequence state for step-wise serving: one *slot* per live request.

A model registers what each of its layer runs keeps per sequence -- a *recurrent* tensor (fixed size: a matrix memory,
a normaliser, a running maximum) or a *row cache* (one row per cached token: keys/values or a compressed latent) -- and
gets back tensors whose first dimension is the slot.  Kernels address a sequence by its slot index, so a step may mix
any slots.  A slot's recurrent tensors are zeroed when it is handed out; its cached rows are simply overwritten from
position 0 (nothing past a sequence's length is ever read).  Freed slots are reused, lowest index first.  ``fork`` gives further requests a
copy of what one holds (answers to the same prompt): one launch for the tensors of all layers.

The reference keeps one static-batch KV cache per generate() call (lia/modeling_opt.py:1379-1491); requests that come and
go need this instead.
"""
import torch

from . import ops


class SlotError(RuntimeError):
    pass


class SlotState:
    def __init__(self, n_slots, capacity, device):
        if n_slots < 1 or capacity < 1:
            raise ValueError("n_slots and capacity must be positive")
        self.n_slots, self.capacity, self.device = int(n_slots), int(capacity), torch.device(device)
        self.recurrent = []                 # tensors [n_slots, ...] zeroed at alloc
        self.rows = []                      # tensors [n_slots, capacity, width], and scales of row caches of 8 and 4 bits
        self.positioned = []                # the same with positions as their second dimension
        self._set = None                    # all of them for copies from slot to slot
        self.length = [0] * self.n_slots    # tokens each slot holds
        self.owner = [None] * self.n_slots
        self.by_id = {}

    # ---- registration (model side)
    def add_recurrent(self, shape, dtype=torch.float32):
        t = torch.zeros((self.n_slots,) + tuple(shape), dtype=dtype, device=self.device)
        self.recurrent.append(t)
        return t

    def add_rows(self, width, dtype):
        t = torch.zeros(self.n_slots, self.capacity, int(width), dtype=dtype, device=self.device)
        self.rows.append(t)
        self.positioned.append(t)
        return t

    def add_rows_8bit(self, heads, dim, dtype):
        """A row cache of ``heads`` heads in int8 or float8_e4m3fn for ``ops.kv_store_8bit``: (codes [n_slots, capacity, heads * dim], scales [n_slots, heads, capacity])."""
        if dtype not in (torch.int8, torch.float8_e4m3fn):
            raise ValueError(f"8-bit rows are int8 or float8_e4m3fn, not {dtype}")
        codes = torch.zeros(self.n_slots, self.capacity, int(heads) * int(dim), dtype=torch.uint8, device=self.device).view(dtype)
        scales = torch.zeros(self.n_slots, int(heads), self.capacity, dtype=torch.float32, device=self.device)
        self.rows += [codes, scales]
        self.positioned += [codes, scales.transpose(1, 2)]
        return codes, scales

    def add_rows_4bit(self, heads, dim):
        """A row cache of ``heads`` heads in 4 bits for ``ops.kv_store_4bit``: (bytes of two codes [n_slots, capacity, heads * dim // 2], bf16 scales [n_slots, heads, capacity, dim // 32])."""
        if dim % 32:
            raise ValueError(f"heads of 4 bits are multiples of 32 channels, not {dim}")
        codes = torch.zeros(self.n_slots, self.capacity, int(heads) * int(dim) // 2, dtype=torch.uint8, device=self.device)
        scales = torch.zeros(self.n_slots, int(heads), self.capacity, int(dim) // 32, dtype=torch.bfloat16, device=self.device)
        self.rows += [codes, scales]
        self.positioned += [codes, scales.transpose(1, 2)]
        return codes, scales

    # ---- requests (scheduler side)
    def slot_of(self, req_id):
        return self.by_id.get(req_id)

    def alloc(self, req_id):
        if req_id in self.by_id:
            raise SlotError(f"request {req_id!r} already holds slot {self.by_id[req_id]}")
        for s in range(self.n_slots):
            if self.owner[s] is None:
                self.owner[s] = req_id
                self.by_id[req_id] = s
                self.length[s] = 0
                for t in self.recurrent:
                    t[s].zero_()
                return s
        raise SlotError(f"all {self.n_slots} slots are in use")

    def fork(self, req_id, new_ids):
        """New requests that go on where ``req_id`` stands: each gets a slot with a copy of its cached rows and recurrent state.  All of them or, where slots or ids do not allow it, none."""
        src, new_ids = self.by_id.get(req_id), list(new_ids)
        if src is None:
            raise SlotError(f"request {req_id!r} holds no slot")
        held = [r for r in new_ids if r in self.by_id]
        if held or len(set(new_ids)) < len(new_ids):
            raise SlotError(f"requests {held or new_ids!r} already hold slots, or are named twice")
        if len(new_ids) > self.owner.count(None):
            raise SlotError(f"{len(new_ids)} slots are needed, {self.owner.count(None)} are free")
        n, to = self.length[src], [s for s in range(self.n_slots) if self.owner[s] is None][:len(new_ids)]
        if self.device.type != "cuda":                                    # (host-resident models: tests)
            for s in to:
                for t in self.recurrent:
                    t[s] = t[src]
                for t in self.positioned:
                    t[s, :n] = t[src, :n]
        elif to and (self.recurrent or self.positioned):
            if self._set is None or len(self._set.tensors) < len(self.positioned) + len(self.recurrent):
                self._set = ops.CacheSet(self.positioned, self.recurrent)
            self._set.fork(torch.tensor([(src, s, n) for s in to], dtype=torch.int32, device=self.device), max_count=n)
        for s, r in zip(to, new_ids):
            self.owner[s], self.length[s], self.by_id[r] = r, n, s
        return to

    def free(self, req_id):
        s = self.by_id.pop(req_id, None)
        if s is None:
            raise SlotError(f"request {req_id!r} holds no slot")
        self.owner[s] = None
        self.length[s] = 0
        return s

    def reserve(self, slot, n):
        """Positions [length, length + n) of ``slot`` for the tokens of this step; returns the first."""
        p0 = self.length[slot]
        if p0 + n > self.capacity:
            raise SlotError(f"slot {slot}: {p0} + {n} tokens exceed the capacity of {self.capacity}")
        self.length[slot] = p0 + n
        return p0

    @property
    def live_tokens(self):
        return sum(self.length)
