"""The attention side without a GPU, continued: what a status word holds, the pool's window, pointers that kernels
would follow to an unaligned address."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sycl-infer_b200", "csrc")


def test_a_bad_page_never_replaces_a_wait_that_ran_out():
    """Both share the prompt kernel's status word.  A wait that runs out is written over whatever is there; a bad page only
    where nothing is: no kernel stores its code unconditionally."""
    for name in ("attn.cuh", "attn_decode.cu", "attn_prompt.cu", "kv.cuh", "kv_pages.cu", "rope_append.cu"):
        text = open(os.path.join(CSRC, name)).read()
        assert not re.search(r"atomic(Exch|Max|Min|Or)\([^;]*B200Q_EINVAL", text), name
    assert re.search(r"note_bad_page\(int \* status\) \{ atomicCAS\(status, 0, B200Q_EINVAL\); \}", open(os.path.join(CSRC, "kv.cuh")).read())
