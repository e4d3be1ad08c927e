"""Host-side mirror of the reference engine's backend-operator interface for the
integer GEMV/GEMM path.

`cuda_backend` carries the same operator names, argument order and meaning as the
reference's `compute_backend` (src/backend/backend.h:33-124 of the reference) for the
operators on this path - `xq`, `i8_gemv`, `i8_gemm`, `gemv_group`, `synchronize` - and
`gemv_seg` mirrors its segment descriptor (src/backend/gpu/kernels/kernels.h:44-81).
Like the reference's backends it is one device + one in-order queue (a CUDA stream),
owns no memory, and raises (RuntimeError subclass) instead of falling back when an
operator is not available.  Buffers are torch CUDA tensors (device memory plumbing
only); every operator goes through the C ABI of libb200q.so.
"""
import ctypes as C
from dataclasses import dataclass
from typing import Optional

import torch

from .attention import _int, _int32
from .capi import MAX_SEGS, AttnOpts, Seg, load_lib


def _ptr(t):
    if t is None:
        return None
    if isinstance(t, int):
        return t
    assert t.is_cuda, "device tensor expected"
    return t.data_ptr()


@dataclass
class gemv_seg:
    """One GEMV output segment (reference: gemv_seg / cpu_gemv_seg)."""
    w: object = None            # uint8 tensor: raw GGUF blocks [n_rows][K]
    type: int = 0               # ggml type id
    K: int = 0
    n_rows: int = 0
    x: object = None            # fp32 activations (fused-quantize operators)
    x_stride: int = 0
    act_up: object = None       # non-None: activation is silu(x)*act_up
    out: object = None          # fp32, out[t*out_stride + row]
    out_stride: int = 0
    residual: object = None
    alpha: float = 1.0
    x8: object = None           # int8 codes, group-major
    xmeta: object = None        # fp32 (scale, 0) pairs
    xsumq: object = None        # int32 pairs of 16-value sums
    i8: bool = True

    def to_c(self):
        return Seg(_ptr(self.w), self.type, self.K, self.n_rows, _ptr(self.x), self.x_stride, _ptr(self.act_up),
                   _ptr(self.out), self.out_stride or self.n_rows, _ptr(self.residual), self.alpha, _ptr(self.x8),
                   _ptr(self.xmeta), _ptr(self.xsumq))


_F32 = torch.float32


def _rows(t, what, index, n_rows, width=None):
    """A 2-D fp32 activation view on CUDA device `index`, one row a token, unit stride within a row: (pointer, row
    stride, row width)."""
    if t.dtype is not _F32 or t.get_device() != index:
        raise ValueError(f"{what}: a float32 tensor on cuda:{index} is expected (got {t.dtype} on {t.device})")
    shape, stride = t.shape, t.stride()
    if len(shape) != 2 or shape[0] != n_rows or (width is not None and shape[1] != width) or (stride[1] != 1 and n_rows):
        raise ValueError(f"{what}: {n_rows} rows" + (f" of {width} values" if width is not None else "") +
                         f" with unit stride are expected (got shape {tuple(shape)}, strides {stride})")
    if stride[0] > 0x7FFFFFFF and n_rows > 1:
        raise ValueError(f"{what}: rows {stride[0]} values apart, 2^31 - 1 at most are supported")
    return t.data_ptr(), stride[0] if n_rows > 1 else shape[1], shape[1]


def _pack(segs):
    if isinstance(segs, gemv_seg):
        segs = [segs]
    if not 1 <= len(segs) <= MAX_SEGS:
        raise ValueError(f"a call holds 1..{MAX_SEGS} segments")
    arr = (Seg * len(segs))(*[s.to_c() for s in segs])
    return arr, len(segs)


class cuda_backend:
    """One B200 + one stream.  Mirrors compute_backend for the int8 GEMV/GEMM path."""

    def __init__(self, device=0, stream: Optional[torch.cuda.Stream] = None):
        if not torch.cuda.is_available():
            raise RuntimeError("cuda_backend needs a CUDA device; this library has no CPU path")
        self.lib = load_lib()
        self.device = torch.device("cuda", device)
        self._stream = stream
        self._attn, self._rope_append = self.lib.attn, self.lib.rope_append

    def name(self):
        return "b200q-cuda"

    def is_cpu(self):
        return False

    def kind(self):
        return "gpu"

    @property
    def stream(self):
        return self._stream if self._stream is not None else torch.cuda.current_stream(self.device)

    def _s(self):
        return C.c_void_p(self.stream.cuda_stream)

    # compute_backend::xq (backend.h:104-105): x8/xmeta/xsumq are caller-owned outputs
    def xq(self, x, up, x_stride, up_stride, x8, xmeta, xsumq, info, TB, K):
        del info  # the reference's host quantizer ignores it as well (xq.cpp:12)
        self.lib.check(self.lib.xq(self._s(), _ptr(x), _ptr(up), x_stride, up_stride, _ptr(x8), _ptr(xmeta),
                                   _ptr(xsumq), TB, K))

    # compute_backend::i8_gemv (backend.h:113); a list runs the segments of one call in one launch
    def i8_gemv(self, s):
        arr, n = _pack(s)
        self.lib.check(self.lib.i8_gemv(self._s(), arr, n))

    # compute_backend::i8_gemm (backend.h:114)
    def i8_gemm(self, s, TB):
        arr, n = _pack(s)
        self.lib.check(self.lib.i8_gemm(self._s(), arr, n, TB))

    # compute_backend::gemv_group (backend.h:61-62): every segment of one type-group of a
    # call, activation given as fp32.  Here the group is quantized into the scratch the
    # segments carry (x8/xmeta/xsumq, engine-owned as in src/engine/graph.cpp:218-220)
    # and run on the integer path; total_rows/nsb/n_tok_blocks are implied by the
    # segments and accepted for signature parity.
    def gemv_group(self, type, segs, n_segs, total_rows, TB, nsb=0, n_tok_blocks=0):
        segs = list(segs)[:n_segs]
        if any(s.type != type for s in segs):
            raise ValueError("gemv_group: every segment must have the group's type")
        if total_rows != sum(s.n_rows for s in segs):
            raise ValueError("gemv_group: total_rows does not match the segments")
        self.quant_gemv(segs, TB)

    # fused decode launch (reference: i8_grp_quant_gemv_launch, kernels.h:216-219)
    def quant_gemv(self, segs, TB=1):
        arr, n = _pack(segs)
        s0 = segs[0] if not isinstance(segs, gemv_seg) else segs
        self.lib.check(self.lib.quant_gemv(self._s(), arr, n, TB, _ptr(s0.x8), _ptr(s0.xmeta), _ptr(s0.xsumq)))

    def quant_gemv_ex(self, segs, TB=1, prequantized=False, peers=None, next_act=None, sync=None, wait=False,
                      signal=False, norm=None, argmax=None):
        """quant_gemv with options: `prequantized` skips the quantizer (the segments' scratch holds
        the activation already); `peers` scatters the outputs; `next_act` = (x8, xmeta, xsumq) makes
        the call emit its output (gate|up: silu(gate)*up) quantized as the following call's activation;
        `sync` = (flag pointer array, world, rank) with `wait` / `signal` folds the cross-GPU flag
        exchange of a row-sharded call into the launch; `norm` = (weight, eps) folds the RMSNorm of
        the activation into the call's quantizer; `argmax` = (idx, val or None) also leaves the row
        index of the largest output (lowest among equals): the LM head of a greedy step."""
        from .capi import ArgmaxOut, CallOpts, NextAct, Norm, PeerSync, OPT_PREQUANTIZED, OPT_SIGNAL_PEERS, OPT_WAIT_PEERS
        arr, n = _pack(segs)
        s0 = segs[0]
        opts = CallOpts()
        opts.flags = (OPT_PREQUANTIZED if prequantized else 0) | (OPT_WAIT_PEERS if wait else 0) | \
            (OPT_SIGNAL_PEERS if signal else 0)
        keep = []
        if peers is not None:
            opts.peers = C.pointer(peers)
        if next_act is not None:
            na = NextAct(_ptr(next_act[0]), _ptr(next_act[1]), _ptr(next_act[2]))
            keep.append(na)
            opts.next = C.pointer(na)
        if argmax is not None:
            am = ArgmaxOut(_ptr(argmax[0]), _ptr(argmax[1]))
            keep.append(am)
            opts.argmax = C.pointer(am)
        if norm is not None:
            nm = Norm(_ptr(norm[0]), float(norm[1]))
            keep.append(nm)
            opts.norm = C.pointer(nm)
        if sync is not None:
            ps = PeerSync(C.cast(sync[0], C.POINTER(C.c_void_p)), sync[1], sync[2])
            keep.append(ps)
            opts.sync = C.pointer(ps)
        self.lib.check(self.lib.quant_gemv_ex(self._s(), arr, n, TB, _ptr(s0.x8), _ptr(s0.xmeta), _ptr(s0.xsumq),
                                              C.byref(opts)))

    def quant_gemv_chain(self, calls):
        """Several dependent one-token calls as one launch where the kernels allow it (same results
        as quant_gemv_ex call by call).  `calls`: a list of (segs, prequantized, next_act)."""
        from .capi import ChainCall, NextAct, OPT_PREQUANTIZED
        arr = (ChainCall * len(calls))()
        keep = []
        for cc, (segs, prequantized, next_act) in zip(arr, calls):
            sa, n = _pack(segs)
            keep.append(sa)
            s0 = segs[0]
            cc.segs, cc.n_segs = sa, n
            cc.x8, cc.xmeta, cc.xsumq = _ptr(s0.x8), _ptr(s0.xmeta), _ptr(s0.xsumq)
            cc.flags = OPT_PREQUANTIZED if prequantized else 0
            if next_act is not None:
                na = NextAct(_ptr(next_act[0]), _ptr(next_act[1]), _ptr(next_act[2]))
                keep.append(na)
                cc.next = C.pointer(na)
        self.lib.check(self.lib.quant_gemv_chain(self._s(), arr, len(calls)))

    # compute_backend::mtp_argmax (backend.h:47-48)
    def mtp_argmax(self, logits, n, out_idx, out_val, M):
        self.lib.check(self.lib.argmax(self._s(), _ptr(logits), n, _ptr(out_idx), _ptr(out_val), M))

    def quant_gemv_scatter(self, segs, TB, peers):
        """quant_gemv whose outputs are also stored into the peers' copies of the output arena."""
        arr, n = _pack(segs)
        s0 = segs[0]
        self.lib.check(self.lib.quant_gemv_scatter(self._s(), arr, n, TB, _ptr(s0.x8), _ptr(s0.xmeta), _ptr(s0.xsumq),
                                                   C.byref(peers)))

    def peer_barrier(self, flag_ptrs, world, rank, seq):
        """Signal every peer that this rank's stores are done and wait for theirs (bounded)."""
        self.lib.check(self.lib.peer_barrier(self._s(), flag_ptrs, world, rank, seq))

    def quant_gemv_static(self, segs):
        """One-token quant_gemv on the library's built-in scratch: for hosts that cannot
        allocate the activation scratch themselves (K <= 32768; calls must not overlap)."""
        arr, n = _pack(segs)
        self.lib.check(self.lib.quant_gemv_static(self._s(), arr, n))

    # ---- attention side: rotary positions + append, attention over the paged cache, page copies ----
    def _here(self, *owners):
        for t in owners:
            if t.device != self.device:
                raise ValueError(f"a tensor on {t.device} was given to the backend of {self.device}")

    def _call(self, fn, *args):
        """fn(stream, *args) with this backend's device current: launches go to the current device's context."""
        index = self.device.index
        stream = self._stream.cuda_stream if self._stream is not None else torch._C._cuda_getCurrentRawStream(index)
        if torch._C._cuda_getDevice() == index:
            rc = fn(stream, *args)
        else:
            with torch.cuda.device(index):
                rc = fn(stream, *args)
        if rc:
            self.lib.check(rc)

    def rope_table(self, rope):
        """Fills rope.table (n_rot / 2 frequencies in turns a position and the factor, 64 bits); once per model."""
        if rope.table is None:
            with torch.cuda.stream(self._stream):  # memory of the stream that writes it (None: the current one)
                rope.table = torch.empty(max(0, rope.c.n_rot) // 2 + 1, dtype=torch.float64, device=self.device)
        self._here(rope.table, *([rope.freq_factors] if rope.freq_factors is not None else []))
        self._call(self.lib.rope_table, rope.ref, rope.table.data_ptr())
        return rope.table

    def rope_append(self, rope, q, k, v, q_out, cache, batch):
        """Rotates q into q_out (may be q itself) and appends the rotated k, and v, to the cache: the newest
        tokens of the batch's sequences.  q, k, v: fp32 rows, views of the q|k|v buffer included; rope None:
        no rotation; q and q_out None: the append alone; k and v None: the rotation of q alone."""
        table = ref = qp = op = kp = vp = None
        qs = os_ = ks = vs = n_head = 0
        self._here(cache, batch)
        if rope is not None:
            if rope.table is None:
                raise ValueError("rope_append: rope_table() has not been called on this rope_t")
            self._here(rope.table)
            table, ref = rope.table.data_ptr(), rope.ref
        if (q is None) != (q_out is None) or (k is None) != (v is None):
            raise ValueError("rope_append: q goes with q_out, k with v")
        index, n = self.device.index, batch.n_tok
        if q is not None:
            qp, qs, width = _rows(q, "rope_append: q", index, n)
            op, os_, _ = _rows(q_out, "rope_append: q_out", index, n, width)
            n_head, odd = divmod(width, cache.head_dim)
            if odd:
                raise ValueError("rope_append: the rows of q are not a multiple of head_dim")
        if k is not None:
            kp, ks, _ = _rows(k, "rope_append: k", index, n, cache.kv_width)
            vp, vs, _ = _rows(v, "rope_append: v", index, n, cache.kv_width)
        if n == 0:
            return
        self._call(self._rope_append, table, ref, qp, qs, n_head, kp, ks, vp, vs, op, os_, cache.ref, batch.ref)

    def attn(self, q, out, cache, batch, scratch, scale=None, window=0, n_sink=0):
        """Attention of the batch's rows over the cache (b200q_attn): causal, with `window` the newest `window` keys
        and the first n_sink ones only.  scratch: attention.alloc_attn_scratch."""
        index, n = self.device.index, batch.n_tok
        self._here(cache, batch, scratch)
        qp, qs, width = _rows(q, "attn: q", index, n)
        op, os_, _ = _rows(out, "attn: out", index, n, width)
        n_head, odd = divmod(width, cache.head_dim)
        if odd:
            raise ValueError("attn: the rows of q are not a multiple of head_dim")
        if not scratch.is_contiguous():
            raise ValueError("attn: the scratch must be contiguous")
        if scale is not None and not C.c_float(scale).value > 0:  # the C side's 0 stands for None
            raise ValueError("attn: scale must be above 0 in 32 bits (None: 1 / sqrt(head_dim))")
        if n == 0:
            return
        opts = AttnOpts(scale or 0.0, window and _int(window, "attn: window"), n_sink and _int(n_sink, "attn: n_sink"))
        self._call(self._attn, qp, qs, n_head, cache.ref, batch.ref, C.byref(opts), op, os_, scratch.data_ptr(), scratch.nbytes)

    def kv_copy_pages(self, caches, src, dst):
        """Page src[i] -> page dst[i] in every cache of the list (the layers of a model): int32 device
        tensors.  dst entries are distinct and none is a src."""
        _int32(src, "kv_copy_pages: src", 1)
        _int32(dst, "kv_copy_pages: dst", 1)
        n = src.numel()
        if n != dst.numel() or not caches:
            raise ValueError("kv_copy_pages: as many dst as src, and at least one cache")
        self._here(src, dst)
        for c in caches:
            if c.index != self.device.index:
                raise ValueError(f"kv_copy_pages: a cache on {c.device} was given to the backend of {self.device}")
        if n:
            self._call(self.lib.kv_copy_pages, b"".join([c.raw for c in caches]), len(caches), src.data_ptr(), dst.data_ptr(), n)

    def kv_remap(self, table, page_map, out=None):
        """out[s][i] = page_map[table[s][i]] (in place without out); entries outside the map stay."""
        out = table if out is None else out
        for t, n, d in ((table, "table", 2), (out, "out", 2), (page_map, "page_map", 1)):
            _int32(t, f"kv_remap: {n}", d)
        n_seq, width = table.shape
        if table.shape != out.shape:
            raise ValueError("kv_remap: out has the table's shape")
        self._here(table, page_map, out)
        if n_seq and width:
            self._call(self.lib.kv_remap, table.data_ptr(), table.stride(0) if n_seq > 1 else width, n_seq, width,
                       page_map.data_ptr(), page_map.numel(), out.data_ptr(), out.stride(0) if n_seq > 1 else width)
        return out

    # parity instrument (no reference operator: the reference never exposes these sums)
    def i8_block_dots(self, w, type, K, n_rows, x8, TB, t, wd):
        self.lib.check(self.lib.i8_block_dots(self._s(), _ptr(w), type, K, n_rows, _ptr(x8), TB, t, _ptr(wd)))

    def device_status(self, clear=True):
        """Error word set by a kernel whose bounded wait ran out (0 = none)."""
        st = C.c_int(0)
        self.lib.check(self.lib.device_status(C.byref(st), 1 if clear else 0))
        return st.value

    # compute_backend::synchronize (backend.h:123): must truly block
    def synchronize(self):
        self.lib.check(self.lib.synchronize(self._s()))


def make_cuda_backend(device=0, stream=None):
    """Counterpart of make_gpu_backend(queue&) (backend.h:126)."""
    return cuda_backend(device, stream)


def alloc_act(TB, K, device="cuda"):
    """Caller-owned quantized-activation scratch of one call (x8, xmeta, xsumq)."""
    G = K // 32
    return (torch.empty(G * TB * 32, dtype=torch.int8, device=device),
            torch.empty(G * TB * 2, dtype=torch.float32, device=device),
            torch.empty(G * TB * 2, dtype=torch.int32, device=device))
