"""The attention side of a decoder layer: paged KV cache, rotary positions, and the pool of pages.

`kv_cache`, `kv_batch` and `rope_t` describe what `cuda_backend.rope_append`, `.attn`, `.kv_copy_pages` and
`.kv_remap` work on; like a `gemv_seg` they hold the caller's tensors and allocate nothing.  `KvPool` is the
host's book of pages: it hands them out, shares them between forked sequences, takes them back and plans the
moves that compact the pool (the roles of the reference's src/engine/engine_kvpool and of the block sharing
in src/engine/engine_prefix_cache).
"""
import ctypes as C
import heapq
import operator
from dataclasses import dataclass, field

import torch

from .capi import KV_TYPES, KvBatch, KvCache, Rope, load_lib

_TORCH_KV = {torch.float16: KV_TYPES["F16"], torch.bfloat16: KV_TYPES["BF16"], torch.float8_e4m3fn: KV_TYPES["E4M3"]}


def _int32(t, what, dims):
    if t.dtype != torch.int32 or t.dim() != dims or not t.is_cuda or (t.numel() and t.stride(-1) != 1):
        raise ValueError(f"{what}: a {dims}-dimensional int32 CUDA tensor with unit stride is expected")


def _int(value, what):
    """An int32 of the C structs, of which ctypes would silently keep the low bits; what is too small the library refuses."""
    if not -2 ** 31 <= value < 2 ** 31:
        raise ValueError(f"{what}: {value} does not fit 32 bits")
    return operator.index(value)  # no fractions


class kv_cache:
    """K and V of one layer: tensors [n_pages][n_kv][page_size][head_dim] of float16, bfloat16 or
    float8_e4m3fn; the pages may lie further apart than they are long (a view of a pool that other layers
    share).  A stored element stands for element * k_scale (v_scale)."""

    def __init__(self, k, v, k_scale=1.0, v_scale=1.0):
        for t, n in ((k, "k"), (v, "v")):
            if t.dim() != 4 or not t.is_cuda or t.dtype not in _TORCH_KV:
                raise ValueError(f"kv_cache: {n} is a CUDA tensor [n_pages][n_kv][page_size][head_dim] of float16, bfloat16 "
                                 "or float8_e4m3fn")
            if t.stride()[1:] != (t.shape[2] * t.shape[3], t.shape[3], 1):
                raise ValueError(f"kv_cache: the pages of {n} must be contiguous in themselves")
        if k.shape != v.shape or k.dtype != v.dtype or k.device != v.device or k.stride() != v.stride():
            raise ValueError("kv_cache: k and v must agree in shape, type, device and strides")
        self.k, self.v, self.device, self.index = k, v, k.device, k.device.index
        self.n_pages, self.n_kv, self.page_size, self.head_dim = k.shape
        self.kv_width = self.n_kv * self.head_dim
        self.c = KvCache(k.data_ptr(), v.data_ptr(), _TORCH_KV[k.dtype], self.n_pages, self.page_size, self.n_kv, self.head_dim,
                         k.stride(0) if self.n_pages > 1 else self.n_kv * self.page_size * self.head_dim, k_scale, v_scale)
        self.ref, self.raw = C.byref(self.c), bytes(self.c)


class kv_batch:
    """The rows of a step (b200q_kv_batch): page_table int32 [n_seq][width], q_start int32 [n_seq + 1],
    kv_len int32 [n_seq].  The kernels read the tensors at every launch, so a recorded step follows what
    the caller writes into them."""

    def __init__(self, page_table, q_start, kv_len, n_tok, max_q):
        _int32(page_table, "kv_batch: page_table", 2)
        _int32(q_start, "kv_batch: q_start", 1)
        _int32(kv_len, "kv_batch: kv_len", 1)
        n_seq = kv_len.numel()
        if n_seq < 1 or q_start.numel() != n_seq + 1 or page_table.shape[0] != n_seq or page_table.shape[1] < 1:
            raise ValueError("kv_batch: n_seq tables, n_seq + 1 row bounds and n_seq lengths are expected")
        if not page_table.device == q_start.device == kv_len.device:
            raise ValueError("kv_batch: tensors on different devices")
        # a table row reaches its own width and no further: rows closer than that would overlap
        stride = page_table.stride(0) if n_seq > 1 else page_table.shape[1]
        if stride != page_table.shape[1]:
            raise ValueError("kv_batch: page_table must be contiguous")
        self.page_table, self.q_start, self.kv_len = page_table, q_start, kv_len
        self.device, self.n_seq = kv_len.device, n_seq
        self.n_tok, self.max_q = _int(int(n_tok), "kv_batch: n_tok"), _int(int(max_q), "kv_batch: max_q")
        self.c = KvBatch(page_table.data_ptr(), q_start.data_ptr(), kv_len.data_ptr(), stride, n_seq, self.n_tok, self.max_q)
        self.ref = C.byref(self.c)


class rope_t:
    """Rotary frequencies (b200q_rope); `cuda_backend.rope_table` fills the table once per model."""

    def __init__(self, n_rot, interleaved=False, base=10000.0, freq_scale=1.0, ext_factor=0.0, attn_factor=1.0, beta_fast=32.0,
                 beta_slow=1.0, n_ctx_orig=0, freq_factors=None):
        if freq_factors is not None and (freq_factors.dtype != torch.float32 or not freq_factors.is_cuda or
                                         not freq_factors.is_contiguous() or freq_factors.numel() != n_rot // 2):
            raise ValueError("rope_t: freq_factors is a contiguous float32 CUDA tensor of n_rot / 2 values")
        self.freq_factors = freq_factors
        self.c = Rope(_int(n_rot, "rope_t: n_rot"), 1 if interleaved else 0, base, freq_scale, ext_factor, attn_factor, beta_fast,
                      beta_slow, _int(n_ctx_orig, "rope_t: n_ctx_orig"), freq_factors.data_ptr() if freq_factors is not None else None)
        self.ref = C.byref(self.c)
        self.table = None  # n_rot / 2 + 1 doubles


def alloc_attn_scratch(n_head, cache, batch):
    """Caller-owned scratch of `cuda_backend.attn`: one serves every layer and step of one stream (how much a call needs
    depends on its shape: take the largest, attn says when it is too small).  It is zeroed when the call returns, for a
    backend on any stream (but for an allocation that is captured: its graph zeroes it).  Calls that may overlap must not
    share it."""
    n = load_lib().attn_scratch_bytes(n_head, cache.n_kv, cache.head_dim, batch.n_seq, batch.n_tok, batch.max_q)
    if n == 0:
        raise ValueError(f"alloc_attn_scratch: unsupported shape ({n_head} heads over {cache.n_kv}, head_dim {cache.head_dim})")
    scratch = torch.zeros(n, dtype=torch.uint8, device=cache.device)
    with torch.cuda.device(cache.device):
        if not torch.cuda.is_current_stream_capturing():
            torch.cuda.current_stream().synchronize()
    return scratch


@dataclass
class attn_call:
    """One layer's attention as a forward plan runs it: q, k, v are the q|k|v call's output (column views of one
    buffer), rotated and appended, then attended; `out` is the o call's activation.  rope None: no positions."""
    q: object
    k: object
    v: object
    out: object
    cache: kv_cache
    batch: kv_batch
    scratch: object
    rope: object = None
    scale: float = None
    window: int = 0
    n_sink: int = 0

    def validate(self, what="attn_call"):
        dim, n_tok = self.cache.head_dim, self.batch.n_tok
        for name, t, width in (("q", self.q, None), ("k", self.k, self.cache.n_kv * dim), ("v", self.v, self.cache.n_kv * dim),
                               ("out", self.out, self.q.shape[1])):
            if t.dim() != 2 or t.shape[0] != n_tok or t.shape[1] != (width or t.shape[1]):
                raise ValueError(f"{what}: {name} has shape {tuple(t.shape)}, {n_tok} rows"
                                 + (f" of {width} values are expected" if width else " are expected"))
        if self.q.shape[1] % (self.cache.n_kv * dim):
            raise ValueError(f"{what}: the query heads are not a multiple of the {self.cache.n_kv} KV heads")
        if self.rope is not None and self.rope.table is None:
            raise ValueError(f"{what}: rope_table() has not been called on the rope_t")

    def run(self, be):
        q = self.q
        be.rope_append(self.rope, q if self.rope is not None else None, self.k, self.v, q if self.rope is not None else None,
                       self.cache, self.batch)
        be.attn(q, self.out, self.cache, self.batch, self.scratch, self.scale, self.window, self.n_sink)


@dataclass
class _Seq:
    pages: list = field(default_factory=list)  # page ids in order, -1 = given back (behind the window)
    length: int = 0                            # tokens
    gone: dict = field(default_factory=dict)   # place of a page given back -> shortest length that does without it
    widest: int = 0                            # window for which pages were given back


class KvPool:
    """Pages of a pool that the layers of a model share (page p of every layer belongs together).

    extend() makes room for a sequence's next tokens and says which pages have to be copied first, because they
    are shared with a fork and about to be written; fork() shares all pages; free() and trim() give pages
    back; compact() plans the moves that bring the pages in use to the front.  The pool owns page numbers only:
    the copies are `cuda_backend.kv_copy_pages`, in the stream in which the step runs.
    """

    def __init__(self, n_pages, page_size):
        if n_pages < 1 or page_size not in (16, 32, 64, 128):
            raise ValueError("KvPool: n_pages >= 1 and a page_size of 16, 32, 64 or 128")
        self.n_pages, self.page_size = int(n_pages), int(page_size)
        self.refs = [0] * self.n_pages
        self._free = list(range(self.n_pages))  # a heap: the lowest page first
        self._seqs, self._next = {}, 0

    @property
    def n_free(self):
        return len(self._free)

    def new(self):
        sid = self._next
        self._next += 1
        self._seqs[sid] = _Seq()
        return sid

    def _seq(self, sid):
        if sid not in self._seqs:
            raise KeyError(f"KvPool: no sequence {sid}")
        return self._seqs[sid]

    def length(self, sid):
        return self._seq(sid).length

    def pages(self, sid):
        return list(self._seq(sid).pages)

    def _take(self):
        p = heapq.heappop(self._free)
        self.refs[p] = 1
        return p

    def _drop(self, p):
        self.refs[p] -= 1
        if self.refs[p] == 0:
            heapq.heappush(self._free, p)

    def extend(self, sid, n):
        """Room for `n` more tokens.  Returns the (src, dst) pairs to copy before they are written: at most the
        sequence's last page, when a fork still holds it.  Raises MemoryError, with nothing changed, when the
        pool has too few pages."""
        q = self._seq(sid)
        if n < 0:
            raise ValueError("KvPool: n >= 0")
        if n == 0:
            return []
        last = q.length // self.page_size  # page that the first new token goes to
        have = len(q.pages)
        # a partly filled last page: written in place unless someone else holds it
        copies = q.length % self.page_size != 0 and q.pages[last] >= 0 and self.refs[q.pages[last]] > 1
        need = -(-(q.length + n) // self.page_size) - have + (1 if copies else 0)
        if need > len(self._free):
            raise MemoryError(f"KvPool: {need} pages wanted, {len(self._free)} free")
        moves = []
        if copies:
            old, new = q.pages[last], self._take()
            self._drop(old)
            q.pages[last] = new
            moves.append((old, new))
        while len(q.pages) * self.page_size < q.length + n:
            q.pages.append(self._take())
        q.length += n
        return moves

    def fork(self, sid):
        """A sequence with the same tokens: every page is shared until one of the two writes to it."""
        q = self._seq(sid)
        for p in q.pages:
            if p >= 0:
                self.refs[p] += 1
        new = self.new()
        self._seqs[new] = _Seq(list(q.pages), q.length, dict(q.gone), q.widest)
        return new

    def truncate(self, sid, length):
        """Forgets the tokens from `length` on (drafts that were not accepted).  Refused, with nothing changed, when the
        window of the next token would reach a page that trim() has given back: truncate first, then trim."""
        q = self._seq(sid)
        if not 0 <= length <= q.length:
            raise ValueError("KvPool: a length within the sequence")
        keep = -(-length // self.page_size)
        first = max(0, (length - q.widest + 1) // self.page_size)  # of the pages that any such window reaches
        if any(q.gone.get(i, 0) > length for i in range(first, keep)):
            raise ValueError(f"KvPool: from token {length} on the window reaches pages that have been given back")
        for i in range(keep, len(q.pages)):
            if q.gone.pop(i, None) is None:
                self._drop(q.pages[i])
        del q.pages[keep:]
        q.length = length

    def trim(self, sid, window, n_sink=0):
        """Gives back the pages that no coming token of a sliding window sees: those wholly behind the window of
        the next token, but for the first n_sink tokens'.  Drafts that may be refused: truncate() comes before trim()."""
        if window < 1 or n_sink < 0:
            raise ValueError("KvPool: window >= 1, n_sink >= 0")
        q = self._seq(sid)
        oldest = q.length - window + 1  # oldest key that the next token, at position `length`, sees
        for i, p in enumerate(q.pages):
            if p >= 0 and (i + 1) * self.page_size <= oldest and i * self.page_size >= n_sink:
                self._drop(p)
                q.pages[i] = -1
                q.gone[i] = (i + 1) * self.page_size + window - 1
                q.widest = max(q.widest, window)

    def free(self, sid):
        q = self._seq(sid)
        for p in q.pages:
            if p >= 0:
                self._drop(p)
        del self._seqs[sid]

    def compact(self):
        """Moves the pages in use to the lowest numbers.  Returns (moves, map): the (src, dst) pairs to copy, no dst of
        which is a src, and every page's new number (for tables that live on the device: `kv_remap`).  The
        sequences' tables change at once."""
        used = [p for p in range(self.n_pages) if self.refs[p] > 0]
        holes = [p for p in range(len(used)) if self.refs[p] == 0]
        moves = list(zip(reversed(used), holes))  # the highest pages fill the lowest holes
        to = dict(moves)
        for a, b in moves:
            self.refs[b], self.refs[a] = self.refs[a], 0
        for q in self._seqs.values():
            q.pages = [to.get(p, p) for p in q.pages]
        self._free = list(range(len(used), self.n_pages))
        return moves, [to.get(p, p) for p in range(self.n_pages)]

    def table(self, sids, width, device="cuda"):
        """Page tables of the sequences, int32 [len(sids)][width], -1 where there is no page."""
        t = torch.full((len(sids), width), -1, dtype=torch.int32)
        for i, s in enumerate(sids):
            p = self._seq(s).pages
            if len(p) > width:
                raise ValueError(f"KvPool: sequence {s} has {len(p)} pages, the table holds {width}")
            if p:
                t[i, :len(p)] = torch.tensor(p, dtype=torch.int32)
        return t.to(device)

    def batch(self, sids, new_tokens, width, device="cuda"):
        """The kv_batch of a step in which sequence sids[i] has just been extended by new_tokens[i]."""
        first = [0]
        for n in new_tokens:
            first.append(first[-1] + int(n))
        i32 = dict(dtype=torch.int32, device=device)
        return kv_batch(self.table(sids, width, device), torch.tensor(first, **i32),
                        torch.tensor([self.length(s) for s in sids], **i32), first[-1], max(1, *map(int, new_tokens)))
