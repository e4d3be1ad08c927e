"""Attention over so many units that a block of the grid (or a warp of it) goes from one to the next: the borders
between units, where shared memory, barriers and tensor memory change hands.  Everything is held to a 64-bit form at
test_gpu_attention.py's tolerance, and repeated calls to the same bits.
"""
import pytest
import torch

from test_gpu_attention import TYPES, split_error

SMS = 148  # blocks of the prompt kernel's grid


# ---- what the kernels share out, by the rules at the head of their files --------------------------------------

def key_tiles(pos_first, n, keys, window, sinks):
    """Tiles of `keys` keys that some row sees, the first of them at position pos_first, of n keys."""
    oldest = min(max(0, pos_first - window + 1) if window else 0, n)
    lo = oldest // keys
    return max(1, min(-(-min(sinks, n) // keys), lo) + -(-n // keys) - lo)


def prompt_units(lens, n_kv, group, window=0, sinks=0):
    """Tiles of every unit (256 rows of a KV head) in the list's order."""
    got = []
    for q, n in lens:
        for r0 in range(0, q * group, 256):
            r1 = min(q * group, r0 + 256) - 1
            got += [key_tiles(n - q + r0 // group, min(n, max(0, n - q + r1 // group + 1)), 128, window, sinks)] * n_kv
    return got


def units_of_blocks(tiles):
    """How many units each block of the prompt kernel works on: equal shares of the list of tiles, three more a unit."""
    total = sum(t + 3 for t in tiles)
    blocks = min(SMS, -(-total // 2))
    each, more = divmod(total, blocks)
    got = []
    for b in range(blocks):
        lo = b * each + min(b, more)
        hi = lo + each + (b < more)
        at = n = 0
        for t in tiles:
            n += min(hi, at + 3 + t) > max(lo, at + 3)
            at += 3 + t
        got.append(n)
    return got


# ---- a step and its 64-bit form ---------------------------------------------------------------------------------

def ragged_step(pkg, typ, lens, n_kv, group, dim, page, seed, window=0, sinks=0, spare=2, q_scale=1.0):
    """(cache, batch, q, first row of each sequence, keys, values): what no row sees is NaN, in the pages too."""
    gen = torch.Generator().manual_seed(seed)
    scales = (0.0625, 0.03125) if typ == "e4m3" else (1.0, 1.0)
    first = [0]
    for q, _ in lens:
        first.append(first[-1] + q)
    held = [-(-n // page) for _, n in lens]
    order = torch.randperm(sum(held) + 2, generator=gen).to(torch.int32)
    pools = [torch.full((sum(held) + 2, n_kv, page, dim), float("nan")) for _ in range(2)]
    table, at, dense = torch.full((len(lens), max(1, *held) + 1), -1, dtype=torch.int32), 0, []
    for s, (q, n) in enumerate(lens):
        j = torch.arange(held[s] * page)
        oldest = max(0, n - q - window + 1) if window and q else 0
        hidden = (j >= n) | ((j < oldest) & (j >= sinks))
        both = []
        for pool, scale in zip(pools, scales):
            x = torch.randn(n_kv, len(j), dim, generator=gen) / scale
            x = x.to(TYPES[typ]).float()
            x[:, hidden] = float("nan")
            pool[order[at:at + held[s]].long()] = x.view(n_kv, held[s], page, dim).transpose(0, 1)
            both.append((x[:, :n] * scale).cuda().double())
        dense.append(both)
        table[s, :held[s]] = order[at:at + held[s]]
        at += held[s]
    n_tok = first[-1] + spare
    q = (q_scale * torch.randn(n_tok, n_kv * group * dim, generator=gen)).cuda()
    cache = pkg.kv_cache(pools[0].to(TYPES[typ]).cuda(), pools[1].to(TYPES[typ]).cuda(), *scales)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    batch = pkg.kv_batch(table.cuda(), i32(first), i32([n for _, n in lens]), n_tok, max(1, *(q for q, _ in lens)))
    return cache, batch, q, first, dense


def reference(cache, batch, q, lens, first, dense, window=0, sinks=0, scale=None):
    """(out, tolerance) in 64 bits; the tolerance is derived at the head of test_gpu_attention.py."""
    dim, kv = cache.head_dim, cache.n_kv
    group = q.shape[1] // dim // kv
    scale = scale or dim ** -0.5
    split = split_error(cache.k.dtype, group * batch.max_q)
    out, tol = (torch.zeros(first[-1], kv, group, dim, dtype=torch.float64, device="cuda") for _ in range(2))
    for s, (n_q, n) in enumerate(lens):
        if not n_q or not n:
            continue
        rows = slice(first[s], first[s] + n_q)
        x = q[rows].double().view(n_q, kv, group, dim)
        pos, j = torch.arange(n - n_q, n, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
        seen = j <= pos
        if window:
            seen &= (j > pos - window) | (j < sinks)
        used = seen.any(0)
        k, v = (t.where(used[None, :, None], torch.zeros_like(t)) for t in dense[s])
        m = seen[:, None, None, :]
        w = torch.softmax(torch.einsum("thgd,hjd->thgj", x, k).mul(scale).masked_fill(~m, float("-inf")), -1)
        w = w.masked_fill(~m, 0.0)  # rows that see nothing: zeros
        out[rows] = torch.einsum("thgj,hjd->thgd", w, v)
        a = torch.einsum("thgd,hjd->thgj", x.abs(), k.abs()).masked_fill(~m, 0.0).amax((1, 2, 3)) * scale
        rel = 2 * a * (split + (dim + 8) * 2.0 ** -24) + split + 2.0 ** -21 + 2 * (n / 16 + 32) * 2.0 ** -24
        top = v.abs().amax(2)[None].where(seen[:, None, :], torch.zeros((), dtype=torch.float64, device="cuda")).amax(2)
        tol[rows] = (rel[:, None] * top)[:, :, None, None]
    return out.flatten(1), tol.flatten(1)


def check(be, pkg, cache, batch, q, lens, first, dense, window=0, sinks=0, scale=None, repeats=1):
    ref, tol = reference(cache, batch, q, lens, first, dense, window, sinks, scale)
    scratch = pkg.alloc_attn_scratch(q.shape[1] // cache.head_dim, cache, batch)
    outs = torch.full((repeats, *q.shape), 77.0, device="cuda")
    for out in outs:
        be.attn(q, out, cache, batch, scratch, scale=scale, window=window, n_sink=sinks)
    be.synchronize()
    n = first[-1]
    assert bool((outs[:, n:] == 77).all()) and be.device_status() == 0
    err = (outs[0, :n].double() - ref).abs()
    assert not bool(err.isnan().any())
    worst = float((err / tol.clamp(min=1e-30)).max())
    assert worst <= 1.0, f"{worst} of the tolerance"
    assert all(torch.equal(out, outs[0]) for out in outs[1:])


# ---- prompts ----------------------------------------------------------------------------------------------------

# (tokens, cache) of the sequences, KV heads, group, window, sinks.  Row blocks end with 1, 20, 33 and 96 live rows (whole
# warps of a tile without any), with more than one tile, and full; units of one tile and of several follow each other.
def _prompts():
    one = [(1, 40), (20, 20), (33, 300), (96, 97), (257, 257), (17, 700), (276, 280), (128, 128), (289, 400), (352, 352)] * 8
    five = [(1, 130), (4, 4), (7, 260), (19, 19), (52, 52), (58, 190), (0, 50), (26, 513)] * 12
    far = [(1, 900), (33, 1000), (20, 20), (129, 640), (5, 3), (97, 97)] * 14
    return {"heads of their own": (one, 8, 1, 0, 0), "groups of five": (five, 8, 5, 0, 0), "window": (far, 8, 4, 70, 4)}


@pytest.mark.parametrize("name", list(_prompts()))
def test_prompt_steps_have_borders(name):
    lens, n_kv, group, window, sinks = _prompts()[name]
    per = units_of_blocks(prompt_units(lens, n_kv, group, window, sinks))
    assert len(per) == SMS and min(per) >= 3, per


@pytest.mark.gpu
@pytest.mark.parametrize("typ", ["bf16", "f16", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("name", list(_prompts()))
def test_prompt_blocks_go_from_unit_to_unit(be, pkg, name, typ, dim):
    lens, n_kv, group, window, sinks = _prompts()[name]
    step = ragged_step(pkg, typ, lens, n_kv, group, dim, 16, seed=dim, window=window, sinks=sinks)
    cache, batch, q, first, dense = step
    check(be, pkg, cache, batch, q, lens, first, dense, window, sinks, repeats=50)


@pytest.mark.gpu
def test_a_wait_lasts_as_long_as_the_block_works(be, pkg):
    """The second row tile's warps have nothing to do in units of up to 128 rows.  4095 sequences of such units over a
    million keys each, then one of 136 rows: they wait for seconds while all is well, and must not give up.  All
    tables name one page, so key j is key j mod 128."""
    n_seq, n_kv, group, dim, page, n, n_q = 4096, 4, 17, 64, 128, 1 << 20, 8
    gen = torch.Generator().manual_seed(1)
    k, v = (torch.randn(1, n_kv, page, dim, generator=gen).to(torch.float16).cuda() for _ in range(2))
    first = torch.arange(n_seq + 1, dtype=torch.int32)
    first[-1] += n_q - 1
    n_tok = n_seq + n_q - 1
    batch = pkg.kv_batch(torch.zeros(n_seq, n // page, dtype=torch.int32, device="cuda"), first.cuda(),
                         torch.full((n_seq,), n, dtype=torch.int32, device="cuda"), n_tok, n_q)
    cache = pkg.kv_cache(k, v)
    q = torch.randn(n_tok, n_kv * group * dim, generator=gen).cuda()
    out = torch.full(q.shape, 77.0, device="cuda")
    be.attn(q, out, cache, batch, pkg.alloc_attn_scratch(n_kv * group, cache, batch))
    be.synchronize()
    assert be.device_status() == 0
    for t, pos in [(0, n - 1), (2000, n - 1)] + [(n_seq - 1 + i, n - n_q + i) for i in range(n_q)]:
        x = q[t].double().view(n_kv, group, dim)
        s = torch.einsum("hgd,hjd->hgj", x, k[0].double()) / 8
        often = (n // page - (torch.arange(page, device="cuda") > pos % page).double()).log()
        want = torch.einsum("hgj,hjd->hgd", torch.softmax(s + often, -1), v[0].double()).flatten()
        a = float(torch.einsum("hgd,hjd->hgj", x.abs(), k[0].double().abs()).max()) / 8
        rel = 2 * a * (2.0 ** -22 + (dim + 8) * 2.0 ** -24) + 2.0 ** -22 + 2.0 ** -21 + 2 * (n / 16 + 32) * 2.0 ** -24
        assert float((out[t].double() - want).abs().max()) <= rel * float(v.abs().max())


# ---- few rows, many units ---------------------------------------------------------------------------------------

# (tokens, cache) of the sequences, KV heads, group, window, sinks: empty slots, sequences without rows and rows before the
# first position among them, units of one tile and units that several warps share.
def _decodes():
    none = [(0, 77), (1, 0), (0, 0), (2, 1)]
    one = ([(1, 1 + 37 * i % 611) for i in range(60)] + none) * 8 + [(1, 9000)]
    some = ([(1 + i % 3, 3 + 53 * i % 700) for i in range(60)] + none) * 8 + [(3, 7000)]
    return {"one row": (one, 8, 4, 0, 0), "up to 15 rows": (some, 8, 5, 0, 0), "window": (some, 8, 4, 90, 5)}


@pytest.mark.parametrize("name", list(_decodes()))
def test_decode_steps_have_borders(name):
    """At most 148 x 3 x 4 warps share the units: two and more for each; and the longest unit alone is more than a warp's share."""
    lens, n_kv, group, window, sinks = _decodes()[name]
    for keys in (16, 32, 64):  # of a tile, by type and head size
        tiles = [key_tiles(n - q, n, keys, window, sinks) for q, n in lens if q]
        assert len(tiles) * n_kv >= 2 * SMS * 3 * 4
        assert window or max(tiles) > sum(tiles) * n_kv / (SMS * 2 * 4)


@pytest.mark.gpu
@pytest.mark.parametrize("typ", ["bf16", "f16", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("name", list(_decodes()))
def test_decode_warps_go_from_unit_to_unit(be, pkg, name, typ, dim):
    lens, n_kv, group, window, sinks = _decodes()[name]
    step = ragged_step(pkg, typ, lens, n_kv, group, dim, 16, seed=dim, window=window, sinks=sinks)
    cache, batch, q, first, dense = step
    check(be, pkg, cache, batch, q, lens, first, dense, window, sinks, repeats=20)


@pytest.mark.gpu
@pytest.mark.parametrize("typ,low", [("bf16", False), ("f16", False), ("e4m3", False), ("bf16", True), ("f16", True), ("e4m3", True)])
@pytest.mark.parametrize("rows", [1, 3, 5])
def test_no_part_of_the_weights_is_lost(be, pkg, typ, low, rows):
    """Few keys and scores near zero: the tolerance is at its smallest, and weights rounded to one 16-bit part, computed
    here in 64 bits, are outside it.  low: many units, few without it; 5 rows x 4 heads go to the prompt kernel."""
    lens = [(rows, rows + 1 + i % 7) for i in range(40 if low else 8)]
    step = ragged_step(pkg, typ, lens, 2, 4, 64, 16, seed=rows)
    cache, batch, q, first, dense = step
    check(be, pkg, cache, batch, q, lens, first, dense, scale=0.004)
    ref, tol = reference(cache, batch, q, lens, first, dense, scale=0.004)
    beyond = 0.0
    for s, (n_q, n) in enumerate(lens):
        x = q[first[s]:first[s] + n_q].double().view(n_q, 2, 4, 64)
        m = torch.arange(n, device="cuda")[None] <= torch.arange(n - n_q, n, device="cuda")[:, None]
        z = torch.einsum("thgd,hjd->thgj", x, dense[s][0]).mul(0.004).masked_fill(~m[:, None, None], float("-inf"))
        p = torch.exp(z - z.amax(-1, keepdim=True))
        one = p.to(torch.bfloat16 if typ == "bf16" else torch.float16).double()
        out = torch.einsum("thgj,hjd->thgd", one / p.sum(-1, keepdim=True), dense[s][1]).flatten(1)
        beyond = max(beyond, float(((out - ref[first[s]:first[s] + n_q]).abs() / tol[first[s]:first[s] + n_q].clamp(min=1e-30)).max()))
    assert beyond > 2.0


# ---- a backend with a stream of its own --------------------------------------------------------------------------

@pytest.mark.gpu
def test_a_scratch_is_ready_for_any_stream(be, pkg):
    """The scratch is zeroed on the caller's stream; the first call on a backend's own stream finds it zeroed, however far
    behind the caller's stream is."""
    lens = [(1, 9000), (1, 30)]
    cache, batch, q, first, dense = ragged_step(pkg, "f16", lens, 2, 4, 64, 16, seed=1)
    ref, tol = reference(cache, batch, q, lens, first, dense)
    own = pkg.make_cuda_backend(0, torch.cuda.Stream())
    first_call = pkg.alloc_attn_scratch(8, cache, batch)
    out = torch.empty(q.shape, device="cuda")
    torch.cuda.synchronize()
    own.attn(q, out, cache, batch, first_call)  # a kernel's first launch may wait for the device
    torch.cuda.synchronize()
    out.fill_(77.0)
    nbytes = first_call.nbytes
    del first_call
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    used = torch.full((nbytes,), 255, dtype=torch.uint8, device="cuda")  # what the allocator hands out again
    torch.cuda.synchronize()
    at = used.data_ptr()
    del used
    torch.cuda._sleep(200_000_000)  # a tenth of a second
    scratch = pkg.alloc_attn_scratch(8, cache, batch)
    assert scratch.data_ptr() == at
    own.attn(q, out, cache, batch, scratch)
    torch.cuda.synchronize()
    assert bool(((out[:2].double() - ref).abs() <= tol).all())


@pytest.mark.gpu
def test_a_rotary_table_is_its_streams_own(be, pkg):
    """The table is written on the backend's stream: its memory must not be some that the caller's stream has yet to write to."""
    want = be.rope_table(pkg.rope_t(128, base=1e6)).clone()
    own = pkg.make_cuda_backend(0, torch.cuda.Stream())
    held = [torch.empty(65, dtype=torch.float64, device="cuda") for _ in range(4200)]  # whatever the allocator has of this size
    torch.cuda.synchronize()
    torch.cuda._sleep(200_000_000)
    held[-1].fill_(7.0)
    held.pop()
    rope = pkg.rope_t(128, base=1e6)
    own.rope_table(rope)
    torch.cuda.synchronize()
    assert torch.equal(rope.table, want)


@pytest.mark.gpu
def test_arguments_beyond_32_bits_are_refused(be, pkg):
    cache, batch, q, first, dense = ragged_step(pkg, "f16", [(1, 40)], 1, 1, 64, 16, seed=1)
    scratch, out = pkg.alloc_attn_scratch(1, cache, batch), torch.empty(q.shape, device="cuda")
    for kw in (dict(window=2 ** 32 + 5), dict(window=2 ** 31), dict(window=5, n_sink=2 ** 32), dict(scale=1e-46), dict(scale=0.0),
               dict(scale=float("nan")), dict(scale=-1.0)):
        with pytest.raises(ValueError):
            be.attn(q, out, cache, batch, scratch, **kw)
    for kw in (dict(window=-1), dict(window=5, n_sink=-1)):
        with pytest.raises(pkg.B200QError):
            be.attn(q, out, cache, batch, scratch, **kw)
    for n_tok, max_q in ((2 ** 32 + 1, 1), (1, 2 ** 32 + 1)):
        with pytest.raises(ValueError):
            pkg.kv_batch(batch.page_table, batch.q_start, batch.kv_len, n_tok, max_q)
    be.attn(q, out, cache, batch, scratch, window=2 ** 31 - 1, n_sink=2 ** 31 - 1, scale=1e-40)
    be.synchronize()
    assert torch.allclose(out[0].double(), dense[0][1][0].mean(0), atol=1e-5, rtol=0)  # no score counts


@pytest.mark.gpu
def test_status_of_kernels_that_have_run(pkg):
    """In a process of its own: the status reads nothing of kernels that have not been launched, and each kernel's bad page
    from its first launch on."""
    import os
    import subprocess
    import sys
    code = """
import torch, __graft_entry__ as graft
pkg = graft.load_package()
be = pkg.make_cuda_backend(0)
assert be.device_status() == 0
i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
pool = torch.zeros(4, 1, 16, 64, dtype=torch.float16, device="cuda")
cache, x, out = pkg.kv_cache(pool, pool.clone()), torch.zeros(20, 64, device="cuda"), torch.zeros(20, 64, device="cuda")
one, many = (pkg.kv_batch(i32([[0, 9]]), i32([0, n]), i32([20]), n, n) for n in (1, 20))
for call in (lambda: be.kv_copy_pages([cache], i32([0]), i32([7])), lambda: be.rope_append(None, None, x[:1], x[:1], None, cache, one),
             lambda: be.attn(x[:1], out[:1], cache, one, pkg.alloc_attn_scratch(1, cache, one)),
             lambda: be.attn(x, out, cache, many, pkg.alloc_attn_scratch(1, cache, many))):
    call()
    be.synchronize()
    assert be.device_status() == 1 and be.device_status() == 0
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run([sys.executable, "-c", code], check=True, cwd=root, timeout=300)


@pytest.mark.gpu
@pytest.mark.parametrize("typ", ["bf16", "e4m3"])
def test_a_recorded_step_of_every_call(be, pkg, typ):
    """Append, prompt and decode attention on one scratch, page copies and the remap, recorded into two graphs that share the
    scratch and run in turn: with other lengths, rows, tables and page lists each time, the bits of the calls one by one."""
    n_kv, group, dim, page, n_tok, n_seq = 2, 5, 64, 16, 160, 3
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    rope = pkg.rope_t(dim, base=1e4)
    be.rope_table(rope)
    qd, kd = n_kv * group * dim, n_kv * dim

    def state():
        gen = torch.Generator().manual_seed(3)
        pools = [torch.randn(64, n_kv, page, dim, generator=gen).to(TYPES[typ]).cuda() for _ in range(2)]
        d = dict(pools=pools, table=torch.zeros(n_seq, 20, dtype=torch.int32, device="cuda"), first=i32([0] * (n_seq + 1)),
                 len=i32([0] * n_seq), one=i32([0, 1, 2, 3]), qkv=torch.zeros(n_tok, qd + 2 * kd, device="cuda"), src=i32([0, 1]),
                 dst=i32([2, 3]), map=torch.arange(64, dtype=torch.int32, device="cuda"), mapped=torch.zeros(n_seq, 20, dtype=torch.int32, device="cuda"),
                 out=torch.zeros(n_tok, qd, device="cuda"), last=torch.zeros(n_seq, qd, device="cuda"), q1=torch.zeros(n_seq, qd, device="cuda"))
        d["cache"] = pkg.kv_cache(*pools)
        d["batch"] = pkg.kv_batch(d["table"], d["first"], d["len"], n_tok, n_tok)
        d["step"] = pkg.kv_batch(d["table"], d["one"], d["len"], n_seq, 1)
        return d

    def run(d, scratch):
        q, k, v = d["qkv"].split([qd, kd, kd], 1)
        be.kv_copy_pages([d["cache"]], d["src"], d["dst"])
        be.rope_append(rope, q, k, v, q, d["cache"], d["batch"])
        be.attn(q, d["out"], d["cache"], d["batch"], scratch, window=70, n_sink=3)
        be.attn(d["q1"], d["last"], d["cache"], d["step"], scratch)
        be.kv_remap(d["table"], d["map"], d["mapped"])

    plain, recorded, again = state(), state(), state()
    scratch = torch.zeros(max(pkg.alloc_attn_scratch(n_kv * group, plain["cache"], plain[b]).nbytes for b in ("batch", "step")), dtype=torch.uint8, device="cuda")
    stream, graphs = torch.cuda.Stream(), []
    torch.cuda.synchronize()
    for d in (recorded, again):
        with torch.cuda.stream(stream):
            run(d, scratch)  # no rows, no keys
            stream.synchronize()
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=stream):
                run(d, scratch)
    run(plain, scratch)  # from here on the three pools are the same: pages 2 and 3 hold what 0 and 1 do
    gen = torch.Generator().manual_seed(4)
    for rows, lens in (([100, 1, 59], [200, 1, 300]), ([0, 160, 0], [16, 160, 0]), ([1, 1, 1], [317, 18, 31]), ([40, 0, 33], [40, 250, 20])):
        pages = torch.randperm(64, generator=gen).to(torch.int32)
        new = dict(table=pages[:60].view(3, 20), len=torch.tensor(lens, dtype=torch.int32), src=pages[60:62], dst=pages[62:64],
                   first=torch.tensor([0, *rows], dtype=torch.int32).cumsum(0, dtype=torch.int32), map=torch.randperm(64, generator=gen).to(torch.int32),
                   qkv=torch.randn(n_tok, qd + 2 * kd, generator=gen), q1=torch.randn(n_seq, qd, generator=gen))
        for d in (plain, recorded, again):
            for name, x in new.items():
                d[name].copy_(x)
            d["out"].fill_(7.0)
        torch.cuda.synchronize()
        run(plain, scratch)
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for d in (recorded, again):
            for name in ("out", "last", "mapped", "qkv"):
                assert torch.equal(d[name], plain[name]), name
            assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(d["pools"], plain["pools"]))
        assert bool((plain["out"][sum(rows):] == 7).all()) and float(plain["last"].abs().max()) > 0
        assert be.device_status() == 0
