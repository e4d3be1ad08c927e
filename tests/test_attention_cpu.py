"""The attention side without a GPU: the pool of pages, and what the entry points refuse (every check is made
on the host, before anything touches a device)."""
import ctypes as C
import random

import pytest

P = 1 << 20  # an aligned address that is never followed: refused calls return before any launch


@pytest.fixture(scope="module")
def capi(pkg):
    from sycl_infer_b200 import capi
    return capi


def cache(capi, **kw):
    d = dict(k=P, v=2 * P, type=30, n_pages=8, page_size=16, n_kv=2, head_dim=64, page_stride=2 * 16 * 64, k_scale=1.0, v_scale=1.0)
    return capi.KvCache(**{**d, **kw})


def batch(capi, **kw):
    d = dict(page_table=P, q_start=P, kv_len=P, table_stride=4, n_seq=2, n_tok=3, max_q=2)
    return capi.KvBatch(**{**d, **kw})


def rope(capi, **kw):
    d = dict(n_rot=64, interleaved=0, base=1e4, freq_scale=1.0, ext_factor=0.0, attn_factor=1.0, beta_fast=32.0, beta_slow=1.0,
             n_ctx_orig=0, freq_factors=None)
    return capi.Rope(**{**d, **kw})


BAD_CACHES = [(dict(k=None), 1), (dict(v=None), 1), (dict(k=P + 8), 1), (dict(type=0), 2), (dict(type=8), 2), (dict(head_dim=96), 2),
              (dict(head_dim=0), 2), (dict(page_size=8), 2), (dict(page_size=48), 2), (dict(n_pages=0), 1), (dict(n_kv=0), 1),
              (dict(page_stride=2 * 16 * 64 - 8), 1), (dict(page_stride=2 * 16 * 64 + 4), 1), (dict(k_scale=0.0), 1),
              (dict(v_scale=-1.0), 1), (dict(k_scale=float("nan")), 1), (dict(v_scale=float("inf")), 1)]
BAD_BATCHES = [dict(page_table=None), dict(q_start=None), dict(kv_len=None), dict(n_seq=0), dict(n_tok=-1), dict(max_q=0), dict(table_stride=0)]


def attn(lib, capi, c=None, b=None, o=None, q=4 * P, qs=256, heads=4, out=8 * P, os_=256, scratch=16 * P, nbytes=1 << 40):
    return lib.attn(None, q, qs, heads, C.byref(c or cache(capi)), C.byref(b or batch(capi)), C.byref(o) if o else None, out, os_, scratch, nbytes)


def append(lib, capi, c=None, b=None, r=None, table=P, q=4 * P, qs=512, heads=4, k=6 * P, ks=128, v=7 * P, vs=128, out=8 * P, os_=256):
    return lib.rope_append(None, table, C.byref(r or rope(capi)), q, qs, heads, k, ks, v, vs, out, os_, C.byref(c or cache(capi)),
                           C.byref(b or batch(capi)))


def test_refused_caches_and_batches(pkg, capi):
    lib = pkg.load_lib()
    for kw, code in BAD_CACHES:
        assert attn(lib, capi, c=cache(capi, **kw)) == code, kw
        assert append(lib, capi, c=cache(capi, **kw)) == code, kw
        arr = (capi.KvCache * 1)(cache(capi, **kw))
        assert lib.kv_copy_pages(None, arr, 1, P, P, 1) == code, kw
        assert lib.last_error()
    for kw in BAD_BATCHES:
        assert attn(lib, capi, b=batch(capi, **kw)) == 1 and append(lib, capi, b=batch(capi, **kw)) == 1, kw


def test_refused_attention(pkg, capi):
    lib = pkg.load_lib()
    for kw in (dict(q=None), dict(out=None), dict(heads=3), dict(heads=0), dict(qs=255), dict(os_=255), dict(scratch=None),
               dict(scratch=16 * P + 4), dict(nbytes=100), dict(out=4 * P), dict(out=4 * P + 1024 - 4), dict(q=4 * P + 2)):
        assert attn(lib, capi, **kw) == 1, kw
        assert "b200q_attn" in lib.last_error()
    for kw in (dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(window=-1), dict(n_sink=-1)):
        assert attn(lib, capi, o=capi.AttnOpts(**kw)) == 1, kw
    need = lib.attn_scratch_bytes(4, 2, 64, 2, 3, 2)
    assert need > 0 and attn(lib, capi, nbytes=need - 1) == 1 and str(need) in lib.last_error()
    for bad in ((4, 3, 64, 1, 1, 1), (4, 2, 80, 1, 1, 1), (0, 1, 64, 1, 1, 1), (4, 2, 64, 0, 1, 1), (4, 2, 64, 1, 1, 0)):
        assert lib.attn_scratch_bytes(*bad) == 0
    assert attn(lib, capi, b=batch(capi, n_seq=4097)) == 2 and "4096" in lib.last_error()
    assert attn(lib, capi, b=batch(capi, n_tok=2 ** 30, max_q=2 ** 30)) == 2
    # no rows: nothing to do, nothing launched
    assert attn(lib, capi, b=batch(capi, n_tok=0)) == 0 and append(lib, capi, b=batch(capi, n_tok=0)) == 0


def test_refused_appends(pkg, capi):
    lib = pkg.load_lib()
    for kw in (dict(q=None, k=None, v=None), dict(k=None), dict(v=None), dict(out=None), dict(qs=255), dict(os_=255), dict(ks=127),
               dict(vs=100), dict(heads=0), dict(table=P + 4), dict(r=rope(capi, n_rot=63)), dict(r=rope(capi, n_rot=0)),
               dict(r=rope(capi, n_rot=66)), dict(r=rope(capi, n_rot=130)), dict(out=4 * P + 4, os_=512), dict(out=6 * P)):
        assert append(lib, capi, **kw) == 1, kw
        assert "b200q_rope_append" in lib.last_error()
    for kw in (dict(n_rot=5), dict(base=1.0), dict(base=float("inf")), dict(freq_scale=0.0), dict(freq_scale=1.5), dict(ext_factor=-1.0),
               dict(ext_factor=1.0), dict(ext_factor=1.0, n_ctx_orig=10, beta_slow=0.0), dict(attn_factor=0.0), dict(base=float("nan"))):
        assert lib.rope_table(None, C.byref(rope(capi, **kw)), P) == 1, kw
    assert lib.rope_table(None, C.byref(rope(capi)), None) == 1


def test_refused_page_operators(pkg, capi):
    lib = pkg.load_lib()
    two = (capi.KvCache * 2)(cache(capi), cache(capi))
    assert lib.kv_copy_pages(None, two, 0, P, P, 1) == 1 and lib.kv_copy_pages(None, two, 2, None, P, 1) == 1
    assert lib.kv_copy_pages(None, two, 2, P, P, -1) == 1 and lib.kv_copy_pages(None, two, 2, None, None, 0) == 0
    assert lib.kv_copy_pages(None, two, 2, P, P, 8) == 1  # eight copies and a source in a pool of eight
    for kw in (dict(n_pages=9), dict(type=1), dict(n_kv=1), dict(page_stride=4096)):
        assert lib.kv_copy_pages(None, (capi.KvCache * 2)(cache(capi), cache(capi, **kw)), 2, P, P, 1) == 1, kw
    ok = (None, P, 8, 2, 8, 2 * P, 4, 3 * P, 8)
    for i, bad in ((1, None), (5, None), (7, None), (2, 7), (8, 7), (3, 0), (4, 0), (6, 0), (7, P + 4)):
        a = list(ok)
        a[i] = bad
        assert lib.kv_remap(*a) == 1, (i, bad)


# ---- the pool -------------------------------------------------------------------------------------------------

class Shadow:
    """The pool's contents as a user sees them: each sequence's tokens, and each page's, by plain lists."""

    def __init__(self, pool):
        self.pool, self.mem, self.seq, self.n = pool, {}, {}, 0

    def copy(self, moves):
        assert len({b for _, b in moves}) == len(moves) and not {a for a, _ in moves} & {b for _, b in moves}
        got = [(b, list(self.mem[a])) for a, b in moves]
        for b, x in got:
            self.mem[b] = x

    def extend(self, s, n):
        self.copy(self.pool.extend(s, n))
        size = self.pool.page_size
        for _ in range(n):
            i = len(self.seq[s])
            page = self.pool.pages(s)[i // size]
            assert self.pool.refs[page] == 1  # a page that is written has one holder
            self.mem.setdefault(page, [None] * size)[i % size] = self.n
            self.seq[s].append(self.n)
            self.n += 1

    def check(self):
        size, held = self.pool.page_size, {}
        for s, tokens in self.seq.items():
            pages = self.pool.pages(s)
            assert self.pool.length(s) == len(tokens) and len(pages) == -(-len(tokens) // size)
            for i, t in enumerate(tokens):
                p = pages[i // size]
                assert p < 0 or self.mem[p][i % size] == t
            for p in pages:
                if p >= 0:
                    held[p] = held.get(p, 0) + 1
        assert [held.get(p, 0) for p in range(self.pool.n_pages)] == self.pool.refs
        assert sorted(self.pool._free) == [p for p in range(self.pool.n_pages) if p not in held]


@pytest.mark.parametrize("seed", range(30))
def test_pool_against_plain_lists(pkg, seed):
    rng = random.Random(seed)
    pool = pkg.KvPool(rng.choice([7, 40]), 16)
    sh = Shadow(pool)
    for _ in range(300):
        what, s = rng.random(), rng.choice(list(sh.seq)) if sh.seq else None
        if s is None or what < 0.1:
            sh.seq[pool.new()] = []
        elif what < 0.6:
            try:
                sh.extend(s, rng.choice([0, 1, 1, 3, 17, 40]))
            except MemoryError:
                pass
        elif what < 0.7:
            sh.seq[pool.fork(s)] = list(sh.seq[s])
        elif what < 0.8:
            pool.free(s)
            del sh.seq[s]
        elif what < 0.86:
            n = rng.randint(max(0, len(sh.seq[s]) - 20), len(sh.seq[s]))
            try:
                pool.truncate(s, n)
                del sh.seq[s][n:]
            except ValueError:
                assert any(p < 0 for p in pool.pages(s))
        elif what < 0.93:
            pool.trim(s, rng.choice([1, 16, 30]), rng.choice([0, 4, 20]))
        else:
            before = {s: pool.pages(s) for s in sh.seq}
            moves, new = pool.compact()
            sh.copy(moves)
            used = pool.n_pages - pool.n_free
            assert all(r > 0 for r in pool.refs[:used])
            for s, pages in before.items():
                assert [new[p] if p >= 0 else p for p in pages] == pool.pages(s)
        sh.check()


def test_trim_keeps_what_the_next_token_sees(pkg):
    pool = pkg.KvPool(10, 16)
    s = pool.new()
    pool.extend(s, 100)
    pool.trim(s, window=37, n_sink=4)
    # the next token, at 100, sees 64..100 and the sinks 0..3
    assert [p >= 0 for p in pool.pages(s)] == [True, False, False, False, True, True, True]
    pool.extend(s, 1)
    pool.trim(s, window=37, n_sink=0)
    assert [p >= 0 for p in pool.pages(s)] == [False] * 4 + [True] * 3
    pool.trim(s, window=1)
    assert [p >= 0 for p in pool.pages(s)] == [False] * 6 + [True]


def test_pool_refusals(pkg):
    for bad in ((0, 16), (4, 10)):
        with pytest.raises(ValueError):
            pkg.KvPool(*bad)
    pool = pkg.KvPool(2, 16)
    s = pool.new()
    pool.extend(s, 20)
    with pytest.raises(MemoryError):
        pool.extend(s, 13)
    assert pool.length(s) == 20 and pool.n_free == 0
    f = pool.fork(s)
    with pytest.raises(MemoryError):
        pool.extend(f, 1)  # the shared last page would have to be copied
    assert pool.pages(f) == pool.pages(s)
    for call in (lambda: pool.extend(s, -1), lambda: pool.truncate(s, 21), lambda: pool.trim(s, 0), lambda: pool.table([s], 1, "cpu")):
        with pytest.raises(ValueError):
            call()
    pool.free(s)
    with pytest.raises(KeyError):
        pool.pages(s)
    assert pool.table([f], 3, "cpu").tolist() == [pool.pages(f) + [-1]]


def test_struct_sizes_match_the_header(tmp_path, capi):
    import os
    import shutil
    import subprocess
    if not shutil.which("gcc"):
        pytest.skip("no gcc")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = [("b200q_kv_cache", capi.KvCache), ("b200q_kv_batch", capi.KvBatch), ("b200q_rope", capi.Rope), ("b200q_attn_opts", capi.AttnOpts)]
    src = '#include <stdio.h>\n#include "b200q.h"\nint main(void) {\n'
    src += "".join(f'  printf("%zu\\n", sizeof({n}));\n' for n, _ in names) + "  return 0;\n}\n"
    (tmp_path / "s.c").write_text(src)
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.join(root, "include"), str(tmp_path / "s.c"), "-o", str(tmp_path / "s")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [C.sizeof(t) for _, t in names]
    assert capi.KV_TYPES == {"F16": 1, "BF16": 30, "E4M3": 256}
