"""The attention side without a GPU, continued: what a status word holds, the pool's window, pointers that kernels
would follow to an unaligned address."""
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
