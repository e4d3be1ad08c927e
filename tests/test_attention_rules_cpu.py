"""The attention side without a GPU, continued: what a status word holds, the pool's window, pointers that kernels
would follow to an unaligned address."""
import ctypes as C
import os
import random
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sycl-infer_b200", "csrc")


def test_a_bad_page_never_replaces_a_wait_that_ran_out():
    """Both share the prompt kernel's status word.  A wait that runs out is written over whatever is there; a bad page only
    where nothing is: no kernel stores its code unconditionally."""
    for name in ("attn.cuh", "attn_decode.cu", "attn_prompt.cu", "kv.cuh", "kv_pages.cu", "rope_append.cu"):
        text = open(os.path.join(CSRC, name)).read()
        assert not re.search(r"atomic(Exch|Max|Min|Or)\([^;]*B200Q_EINVAL", text), name
    assert re.search(r"note_bad_page\(int \* status\) \{ atomicCAS\(status, 0, B200Q_EINVAL\); \}", open(os.path.join(CSRC, "kv.cuh")).read())


def _needed(length, window, sinks, size):
    """Pages that the token at position `length` needs: those of the keys that it sees, and the one that it is written to
    when tokens before it have begun it."""
    return {j // size for j in range(length) if j > length - window or j < sinks} | ({length // size} if length % size else set())


def test_truncate_keeps_what_the_next_token_sees(pkg):
    pool = pkg.KvPool(10, 16)
    s = pool.new()
    pool.extend(s, 100)
    pool.trim(s, 37)  # pages below key 64
    before = pool.pages(s)
    for n in (95, 99, 64, 70, 1):  # from 95 the next token sees 59 .. 95
        with pytest.raises(ValueError, match="given back"):
            pool.truncate(s, n)
    assert pool.pages(s) == before and pool.length(s) == 100
    f = pool.fork(s)
    with pytest.raises(ValueError):
        pool.truncate(f, 99)
    pool.truncate(f, 0)  # nothing before it: nothing that is gone
    assert pool.pages(f) == []
    pool.extend(s, 12)
    pool.truncate(s, 100)
    pool.trim(s, 1)
    pool.truncate(s, 100)
    assert pool.length(s) == 100


@pytest.mark.parametrize("seed", range(20))
def test_pages_in_the_window_survive_trim_and_truncate(pkg, seed):
    """A drafting loop in any order: every key that the window of the next token holds has its page, and a refused
    truncation is one after which some key would not."""
    rng = random.Random(seed)
    size = rng.choice([16, 32])
    pool = pkg.KvPool(60, size)
    window, sinks, s = rng.choice([1, 16, 37, 100]), rng.choice([0, 4, 20]), pool.new()
    for _ in range(400):
        what = rng.random()
        if what < 0.5 and pool.length(s) < 40 * size:
            pool.extend(s, rng.choice([1, 2, 5, 30]))
        elif what < 0.75:
            pool.trim(s, window, sinks)
        else:
            n, before = rng.randint(max(0, pool.length(s) - 40), pool.length(s)), pool.pages(s)
            lost = any(before[i] < 0 for i in _needed(n, window, sinks, size))
            if lost:
                with pytest.raises(ValueError):
                    pool.truncate(s, n)
                assert pool.pages(s) == before
            else:
                pool.truncate(s, n)
        assert all(pool.pages(s)[i] >= 0 for i in _needed(pool.length(s), window, sinks, size))


def test_unaligned_pointers_are_refused(pkg):
    """No entry point hands a kernel an address that its loads and stores would fault on."""
    from sycl_infer_b200 import capi
    lib, P = pkg.load_lib(), 1 << 20

    def cache():
        return capi.KvCache(P, 2 * P, 30, 8, 16, 2, 64, 2 * 16 * 64, 1.0, 1.0)

    def batch(**kw):
        d = dict(page_table=P, q_start=P, kv_len=P, table_stride=4, n_seq=2, n_tok=3, max_q=2)
        return C.byref(capi.KvBatch(**{**d, **kw}))

    def rope(**kw):
        return C.byref(capi.Rope(**{**dict(n_rot=64, base=1e4, freq_scale=1.0, attn_factor=1.0, beta_fast=32.0, beta_slow=1.0), **kw}))

    def append(b=None, q=4 * P, k=6 * P, v=7 * P, out=8 * P):
        return lib.rope_append(None, P, rope(), q, 512, 4, k, 128, v, 128, out, 256, C.byref(cache()), b or batch())

    def attn(b=None, q=4 * P, out=8 * P):
        return lib.attn(None, q, 256, 4, C.byref(cache()), b or batch(), None, out, 256, 16 * P, 1 << 40)

    for off in (1, 2, 3):
        for name in ("page_table", "q_start", "kv_len"):
            assert append(batch(**{name: P + off})) == 1 and attn(batch(**{name: P + off})) == 1, name
            assert "aligned" in lib.last_error()
        for name, base in (("q", 4 * P), ("k", 6 * P), ("v", 7 * P), ("out", 8 * P)):
            assert append(**{name: base + off}) == 1, name
        assert attn(q=4 * P + off) == 1 and attn(out=8 * P + off) == 1
        assert lib.rope_table(None, rope(freq_factors=P + off), P) == 1
        arr = (capi.KvCache * 1)(cache())
        assert lib.kv_copy_pages(None, arr, 1, P + off, P, 1) == 1 and lib.kv_copy_pages(None, arr, 1, P, P + off, 1) == 1
        for i in (1, 5, 7):
            a = [None, P, 8, 2, 8, 2 * P, 4, 3 * P, 8]
            a[i] += off
            assert lib.kv_remap(*a) == 1, i


def test_counts_beyond_32_bits_are_refused(pkg):
    """Not cut to their low 32 bits."""
    import torch
    from sycl_infer_b200.backend import _rows
    for kw in (dict(n_rot=2 ** 32 + 64), dict(n_rot=64, n_ctx_orig=2 ** 32 + 4096)):
        with pytest.raises(ValueError):
            pkg.rope_t(**kw)

    with pytest.raises(TypeError):
        pkg.rope_t(64.5)

    class view:  # rows that far apart take more memory than there is
        dtype, shape = torch.float32, (2, 256)
        get_device, data_ptr = (lambda self: 0), (lambda self: 1 << 20)

        def __init__(self, apart):
            self.apart = apart

        def stride(self):
            return self.apart, 1

    assert _rows(view(2 ** 31 - 1), "q", 0, 2) == (1 << 20, 2 ** 31 - 1, 256)
    for apart in (2 ** 31, 2 ** 32 + 256):
        with pytest.raises(ValueError, match="apart"):
            _rows(view(apart), "q", 0, 2)
