"""Rotary append, paged attention and page operators against plain 64-bit forms.

Attention's tolerance, element by element (natural exponent, a = largest scale * sum_d |q_d k_d|):
a score is off by at most a * (s + (D + 8) 2^-24): s from splitting q into 16-bit parts, each of which leaves half a step
(fp16 2^-11, bf16 2^-8) of what the part before it left: 2^-22 for two fp16 parts (fp16 and e4m3 caches), 2^-24 for the three bf16
parts of up to 16 query rows a KV head, 2^-16 for the two of more rows; the rest from fp32 sums over D products and the two roundings of the
scaling; relative weights by twice that (numerator and sum), plus s again for the split of the weights, plus 2^-21
for ex2.approx (2^-22, numerator and sum), plus fp32 sums over n keys, which run in chains of n / 16 + 32 at most.
The output is a weighted mean of v, so it is off by at most that times the largest |v| of its head.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}


def make_step(pkg, typ, lens, n_kv, group, dim, page, seed=0, window=0, sinks=0, spare=2, scales=(1.0, 1.0), held=True):
    """A cache in which only the visible keys hold numbers and everything else is NaN, and a step's rows.
    lens: (new tokens, cache length) a sequence.  Pages nobody sees are not in the table (-1)."""
    gen = torch.Generator().manual_seed(seed)
    first = [0]
    for q, _ in lens:
        first.append(first[-1] + q)
    n_tok = first[-1] + spare
    width = max(1, max(-(-n // page) for _, n in lens)) + 1
    need = []
    for q, n in lens:
        oldest = max(0, n - q - window + 1) if window else 0
        need.append([p for p in range(-(-n // page)) if (p + 1) * page > oldest or p * page < sinks])
    n_pages = sum(map(len, need)) + 2
    order = torch.randperm(n_pages, generator=gen).to(torch.int32)
    table, at = torch.full((len(lens), width), -1, dtype=torch.int32), 0
    k = torch.full((n_pages, n_kv, page, dim), float("nan"))
    v = k.clone()
    for s, (q, n) in enumerate(lens):
        oldest = max(0, n - q - window + 1) if window else 0
        for p in need[s]:
            table[s, p] = order[at]
            for t in range(page):
                j = p * page + t
                if held and j < n and (j >= oldest or j < sinks):
                    k[order[at], :, t] = torch.randn(n_kv, dim, generator=gen) / scales[0]
                    v[order[at], :, t] = torch.randn(n_kv, dim, generator=gen) / scales[1]
            at += 1
    qd = n_kv * group * dim
    buf = torch.randn(n_tok, qd + 24, generator=gen).cuda()
    cache = pkg.kv_cache(k.to(TYPES[typ]).cuda(), v.to(TYPES[typ]).cuda(), *scales)
    max_q = max(q for q, _ in lens) or 1
    batch = pkg.kv_batch(table.cuda(), torch.tensor(first, dtype=torch.int32).cuda(),
                         torch.tensor([n for _, n in lens], dtype=torch.int32).cuda(), n_tok, max_q)
    return cache, batch, buf[:, 4:4 + qd], first


def dense(pool, table, n, page, scale):
    """Keys or values 0..n-1 of one sequence in 64 bits, [n_kv][n][dim]; NaN where there is no page."""
    x = pool.to(torch.float32) if pool.dtype == torch.float8_e4m3fn else pool
    j = torch.arange(n, device=pool.device)
    p = table.long()[j // page]
    got = x[p.clamp(min=0)[:, None], torch.arange(pool.shape[1], device=pool.device)[None], (j % page)[:, None]].double() * scale
    got[p < 0] = float("nan")
    return got.transpose(0, 1)


def split_error(dtype, rows):
    return 2.0 ** -22 if dtype != torch.bfloat16 else (2.0 ** -24 if rows <= 16 else 2.0 ** -16)


def attn_ref(cache, batch, q, lens, first, window, sinks, scale):
    """(out, tolerance) in 64 bits, one row and head at a time over the keys that it sees."""
    n_tok, qd = q.shape
    dim, page = cache.head_dim, cache.page_size
    group = qd // dim // cache.n_kv
    out = torch.zeros(n_tok, qd, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    split = split_error(cache.k.dtype, group * batch.max_q)
    for s, (n_q, n) in enumerate(lens):
        if n == 0:
            continue
        k, v = dense(cache.k, batch.page_table[s], n, page, cache.c.k_scale), dense(cache.v, batch.page_table[s], n, page, cache.c.v_scale)
        for i in range(n_q):
            pos = n - n_q + i
            j = torch.arange(n, device="cuda")
            seen = j <= pos
            if window:
                seen &= (j > pos - window) | (j < sinks)
            if not bool(seen.any()):
                continue
            kk, vv = k[:, seen].repeat_interleave(group, 0), v[:, seen].repeat_interleave(group, 0)
            x = q[first[s] + i].double().view(-1, 1, dim)
            w = torch.softmax((x * kk).sum(-1) * scale, -1)
            out[first[s] + i] = (w[:, :, None] * vv).sum(1).flatten()
            a = float((x * kk).abs().sum(-1).max()) * scale
            rel = 2 * a * (split + (dim + 8) * 2.0 ** -24) + split + 2.0 ** -21 + 2 * (n / 16 + 32) * 2.0 ** -24
            tol[first[s] + i] = (vv.abs().amax((1, 2)) * rel)[:, None].expand(-1, dim).flatten()
    return out, tol


def check_attn(be, pkg, cache, batch, q, lens, first, window=0, sinks=0, scale=None, scratch=None):
    wide = torch.full((q.shape[0], q.shape[1] + 8), 77.0, device="cuda")
    out = wide[:, 4:4 + q.shape[1]]
    scratch = pkg.alloc_attn_scratch(q.shape[1] // cache.head_dim, cache, batch) if scratch is None else scratch
    be.attn(q, out, cache, batch, scratch, scale=scale, window=window, n_sink=sinks)
    be.synchronize()
    ref, tol = attn_ref(cache, batch, q, lens, first, window, sinks, scale or cache.head_dim ** -0.5)
    used = first[-1]
    assert bool((wide[used:] == 77).all()) and bool((wide[:, :4] == 77).all()) and bool((wide[:, -4:] == 77).all())
    err = (out[:used].double() - ref[:used]).abs()
    assert not bool(err.isnan().any())
    worst = float((err / tol[:used].clamp(min=1e-30)).max())
    assert worst <= 1.0, f"{worst} of the tolerance"
    assert be.device_status() == 0


@pytest.mark.parametrize("typ", ["bf16", "f16", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n_kv,group", [(1, 1), (2, 5), (3, 8), (2, 16), (1, 3)])
def test_decode_types_and_heads(be, pkg, typ, dim, n_kv, group):
    lens = [(1, 1), (1, 77), (1, 300), (1, 16)]
    scales = (0.0625, 0.03125) if typ == "e4m3" else (1.0, 1.0)
    cache, batch, q, first = make_step(pkg, typ, lens, n_kv, group, dim, 16, scales=scales)
    check_attn(be, pkg, cache, batch, q, lens, first)


@pytest.mark.parametrize("typ", ["bf16", "f16", "e4m3"])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("n", [1, 15, 16, 17, 63, 64, 65, 127, 129, 1000, 4097])
def test_decode_lengths(be, pkg, typ, page, n):
    lens = [(1, n)]
    cache, batch, q, first = make_step(pkg, typ, lens, 2, 4, 64, page, seed=n)
    check_attn(be, pkg, cache, batch, q, lens, first, scale=0.2)


@pytest.mark.parametrize("typ", ["bf16", "e4m3"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (33, 0), (100, 130), (64, 20), (5000, 3)])
def test_window_and_sinks(be, pkg, typ, window, sinks):
    lens = [(1, 500), (1, 20), (3, 777), (1, 1), (2, 130)]
    cache, batch, q, first = make_step(pkg, typ, lens, 2, 3, 128, 16, seed=window, window=window, sinks=sinks)
    check_attn(be, pkg, cache, batch, q, lens, first, window, sinks)


@pytest.mark.parametrize("typ", ["bf16", "f16", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens", [[(7, 7)], [(33, 33), (2, 90), (70, 200)], [(130, 131), (1, 400), (64, 64)], [(300, 300)],
                                  [(257, 600), (5, 5)]])
def test_several_tokens(be, pkg, typ, dim, lens):
    cache, batch, q, first = make_step(pkg, typ, lens, 2, 5, dim, 32, seed=3)
    check_attn(be, pkg, cache, batch, q, lens, first)


@pytest.mark.parametrize("typ", ["bf16", "e4m3"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (20, 0), (50, 4), (200, 140)])
def test_several_tokens_in_a_window(be, pkg, typ, window, sinks):
    lens = [(150, 400), (1, 30), (90, 90), (40, 300)]
    cache, batch, q, first = make_step(pkg, typ, lens, 1, 4, 64, 16, seed=window, window=window, sinks=sinks)
    check_attn(be, pkg, cache, batch, q, lens, first, window, sinks)


@pytest.mark.parametrize("lens", [[(1, 0)], [(0, 0), (1, 40), (0, 64), (1, 0), (1, 5)], [(1, 0)] * 3 + [(2, 300)], [(3, 2)], [(40, 25), (1, 9)]])
def test_rows_that_see_nothing(be, pkg, lens):
    """Empty slots, sequences without rows, and rows before the first position give zeros (or nothing)."""
    cache, batch, q, first = make_step(pkg, "bf16", lens, 2, 4, 64, 16)
    check_attn(be, pkg, cache, batch, q, lens, first)


def test_many_sequences(be, pkg):
    lens = [(1, 1 + 13 * i % 97) for i in range(301)]
    cache, batch, q, first = make_step(pkg, "f16", lens, 2, 2, 64, 16)
    check_attn(be, pkg, cache, batch, q, lens, first)


def test_large_scores_and_values(be, pkg):
    """One key far above the others, scores of either sign in the hundreds, large values: nothing overflows."""
    lens = [(1, 200), (2, 64)]
    for typ in ("bf16", "f16"):
        cache, batch, q, first = make_step(pkg, typ, lens, 2, 4, 128, 16)
        q.mul_(30.0)
        cache.v.mul_(1000.0)
        check_attn(be, pkg, cache, batch, q, lens, first)


@pytest.mark.parametrize("lens", [[(1, 300), (1, 77)], [(60, 60), (3, 200)]])
@pytest.mark.parametrize("typ", ["f16", "e4m3"])
def test_unaligned_rows(be, pkg, typ, lens):
    """Rows of q and out that start off 16 bytes and lie an odd number of values apart."""
    cache, batch, q, first = make_step(pkg, typ, lens, 2, 3, 64, 16)
    wide = torch.randn(q.shape[0], q.shape[1] + 3, device="cuda")
    view = wide[:, 1:1 + q.shape[1]]
    out = torch.zeros(q.shape[0], q.shape[1] + 5, device="cuda")[:, 3:3 + q.shape[1]]
    be.attn(view, out, cache, batch, pkg.alloc_attn_scratch(6, cache, batch))
    ref, tol = attn_ref(cache, batch, view, lens, first, 0, 0, 64 ** -0.5)
    n = first[-1]
    assert bool(((out[:n].double() - ref[:n]).abs() <= tol[:n]).all()) and bool((out[n:] == 0).all())


@pytest.mark.parametrize("group,lens", [(1, [(40, 70), (20, 20)]), (17, [(1, 90), (2, 33)]), (40, [(1, 200)]), (300, [(3, 50)]), (7, [(19, 400), (37, 37)])])
def test_prompt_groups(be, pkg, group, lens):
    """Head groups that do not divide the row tiles, larger than one among them."""
    cache, batch, q, first = make_step(pkg, "f16", lens, 1, group, 64, 16)
    check_attn(be, pkg, cache, batch, q, lens, first)


def test_rows_beyond_max_q_are_left(be, pkg):
    for n_q, max_q in ((5, 2), (60, 40)):
        lens = [(n_q, 100)]
        cache, batch, q, first = make_step(pkg, "f16", lens, 1, 4, 64, 16)
        short = pkg.kv_batch(batch.page_table, batch.q_start, batch.kv_len, batch.n_tok, max_q)
        out = torch.full(q.shape, 5.0, device="cuda")
        be.attn(q, out, cache, short, pkg.alloc_attn_scratch(4, cache, short))
        ref, tol = attn_ref(cache, short, q, lens, first, 0, 0, 64 ** -0.5)
        assert bool(((out[:max_q].double() - ref[:max_q]).abs() <= tol[:max_q]).all()) and bool((out[max_q:] == 5).all())


def test_a_window_without_end(be, pkg):
    """The largest window and sink count are no window at all."""
    for lens in ([(1, 700)], [(50, 300)]):
        cache, batch, q, first = make_step(pkg, "bf16", lens, 1, 4, 64, 16)
        check_attn(be, pkg, cache, batch, q, lens, first, 2 ** 31 - 1, 2 ** 31 - 1)


def test_one_scratch_for_calls_of_all_shapes(be, pkg):
    """Decode and prompt steps of few and of many sequences take turns on one scratch: none finds another's leavings."""
    steps = []
    for lens, kv, group, dim, typ in ([(1, 5000)], 2, 4, 64, "bf16"), ([(1, 40 + i) for i in range(150)], 2, 4, 128, "f16"), \
            ([(300, 900), (40, 2000)], 2, 8, 128, "f16"), ([(3, 3000)] * 3, 1, 5, 128, "bf16"), ([(100, 100)] * 5, 2, 4, 64, "e4m3"):
        cache, batch, q, first = make_step(pkg, typ, lens, kv, group, dim, 16)
        ref, tol = attn_ref(cache, batch, q, lens, first, 0, 0, dim ** -0.5)
        need = pkg.load_lib().attn_scratch_bytes(kv * group, kv, dim, batch.n_seq, batch.n_tok, batch.max_q)
        steps.append((cache, batch, q, first[-1], ref, tol, need))
    scratch = torch.zeros(max(s[-1] for s in steps), dtype=torch.uint8, device="cuda")
    for turn in range(4):
        for cache, batch, q, n, ref, tol, _ in (steps if turn % 2 else steps[::-1]):
            out = torch.empty(q.shape, device="cuda")
            be.attn(q, out, cache, batch, scratch)
            assert bool(((out[:n].double() - ref[:n]).abs() <= tol[:n]).all())
    assert bool((scratch[:8192] == 0).all())


def test_two_streams_at_once(be, pkg):
    """Calls on two streams, each with a scratch of its own, do not disturb each other."""
    backs, runs = [pkg.make_cuda_backend(0, torch.cuda.Stream()) for _ in range(2)], []
    for b, lens in zip(backs, ([(1, 9000), (1, 30)], [(130, 700), (9, 9)])):
        cache, batch, q, first = make_step(pkg, "f16", lens, 2, 4, 64, 16)
        ref, tol = attn_ref(cache, batch, q, lens, first, 0, 0, 64 ** -0.5)
        runs.append((b, cache, batch, q, first[-1], ref, tol, pkg.alloc_attn_scratch(8, cache, batch), [torch.zeros(q.shape, device="cuda") for _ in range(12)]))
    torch.cuda.synchronize()
    for i in range(12):
        for b, cache, batch, q, n, ref, tol, scratch, outs in runs:
            b.attn(q, outs[i], cache, batch, scratch)
    torch.cuda.synchronize()
    for b, cache, batch, q, n, ref, tol, scratch, outs in runs:
        for out in outs:
            assert bool(((out[:n].double() - ref[:n]).abs() <= tol[:n]).all())


def test_a_pool_beyond_4_gb(be, pkg):
    """Pages whose byte offsets pass 32 bits: append, both attentions and the page copy reach them."""
    n_pages, page, dim = 9, 16, 64
    mem = torch.empty(2, n_pages, 1 << 28, dtype=torch.bfloat16, device="cuda")  # 512 MB from page to page
    k, v = (m[:, :2 * page * dim].view(n_pages, 2, page, dim) for m in mem)
    k.zero_()
    v.zero_()
    cache = pkg.kv_cache(k, v)
    table = torch.tensor([[8, 0, 7]], dtype=torch.int32).cuda()
    n = 40
    batch = pkg.kv_batch(table, torch.tensor([0, n], dtype=torch.int32).cuda(), torch.tensor([n], dtype=torch.int32).cuda(), n, n)
    x = torch.randn(n, 8 * dim, device="cuda")
    q, kn, vn = x.split([4 * dim, 2 * dim, 2 * dim], 1)
    be.rope_append(None, None, kn, vn, None, cache, batch)
    for i in range(n):
        p, at = int(table[0, i // page]), i % page
        assert torch.equal(k[p, :, at].flatten(), kn[i].bfloat16()) and torch.equal(v[p, :, at].flatten(), vn[i].bfloat16())
    lens = [(n, n)]
    check_attn(be, pkg, cache, batch, q, lens, [0, n])
    one = pkg.kv_batch(table, torch.tensor([0, 1], dtype=torch.int32).cuda(), batch.kv_len, 1, 1)
    check_attn(be, pkg, cache, one, q[:1], [(1, n)], [0, 1])
    be.kv_copy_pages([cache], torch.tensor([8, 0], dtype=torch.int32).cuda(), torch.tensor([1, 6], dtype=torch.int32).cuda())
    assert torch.equal(k[1], k[8]) and torch.equal(v[6], v[0])


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("k_size,v_size", [(1.0, 1e-7), (1.0, 3e9), (2e6, 1.0), (1e-9, 1e-20), (1e20, 1e30), (1.0, 0.0)])
def test_bf16_prompts_of_any_magnitude(be, pkg, dim, k_size, v_size):
    """Keys and values far outside fp16's range, unequal from page to page: bf16 has it."""
    lens = [(60, 400), (33, 33)]
    cache, batch, q, first = make_step(pkg, "bf16", lens, 2, 4, dim, 16)
    cache.k.mul_(k_size)
    cache.v.mul_(v_size)
    cache.v[1::3].mul_(0.001)  # and unequal from page to page
    q.mul_(1.0 / k_size)
    check_attn(be, pkg, cache, batch, q, lens, first)


def test_results_do_not_depend_on_arrival(be, pkg):
    lens = [(1, 20000), (1, 3000), (1, 50)]
    cache, batch, q, first = make_step(pkg, "bf16", lens, 2, 4, 64, 64)
    scratch = pkg.alloc_attn_scratch(8, cache, batch)
    out = torch.empty(q.shape, device="cuda")
    be.attn(q, out, cache, batch, scratch)
    one = out.clone()
    for _ in range(20):
        out.zero_()
        be.attn(q, out, cache, batch, scratch)
        assert torch.equal(one[:3], out[:3])


def test_captured_step_follows_lengths(be, pkg):
    """A recorded launch serves other lengths, tables and rows later; the scratch is ready for the next call."""
    lens = [(1, 900), (1, 33)]
    cache, batch, q, first = make_step(pkg, "bf16", lens, 2, 4, 64, 16)
    q = q.clone()
    out = torch.zeros(q.shape, device="cuda")
    scratch = pkg.alloc_attn_scratch(8, cache, batch)
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        be.attn(q, out, cache, batch, scratch)
        st.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            be.attn(q, out, cache, batch, scratch)
    for now in ([(1, 900), (1, 33)], [(1, 1), (1, 30)], [(1, 417), (1, 0)], [(1, 899), (1, 2)]):
        batch.kv_len.copy_(torch.tensor([n for _, n in now], dtype=torch.int32))
        out.fill_(5.0)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        ref, tol = attn_ref(cache, batch, q, now, first, 0, 0, 64 ** -0.5)
        assert bool(((out[:2].double() - ref[:2]).abs() <= tol[:2]).all())
        assert bool((out[2:] == 5.0).all())


@pytest.mark.parametrize("n_q", [1, 40])
def test_bad_pages_are_left_out(be, pkg, n_q):
    """A page id outside the pool: its keys are left out, the status says so, nothing is read out of bounds."""
    lens = [(n_q, 100)]
    cache, batch, q, first = make_step(pkg, "bf16", lens, 1, 4, 64, 16)
    assert be.device_status() == 0
    good = batch.page_table.clone()
    for bad in (-1, -7, cache.n_pages, 2 ** 31 - 1):
        batch.page_table.copy_(good)
        batch.page_table[0, 2] = bad
        out = torch.zeros(q.shape, device="cuda")
        be.attn(q, out, cache, batch, pkg.alloc_attn_scratch(4, cache, batch))
        be.synchronize()
        assert be.device_status() == 1 and be.device_status() == 0
        k, v = (dense(p, good[0], 100, 16, 1.0)[0] for p in (cache.k, cache.v))
        keep = [j for j in range(100) if not 32 <= j < 48]
        for i in (0, n_q - 1):
            js = [j for j in keep if j <= 100 - n_q + i]
            w = torch.softmax(q[i].double().view(4, 64) @ k[js].T / 8, -1)
            assert torch.allclose(out[i].double().view(4, 64), w @ v[js], atol=1e-4, rtol=0)


# ---- rotary append ------------------------------------------------------------------------------------------

def rope_ref(x, pos, turns, factor, n, interleaved):
    """x [heads][dim] in 64 bits."""
    x = x.double().clone()
    i = torch.arange(n // 2, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n // 2)
    phase = 2 * math.pi * torch.remainder(pos * turns, 1.0)
    c, s = torch.cos(phase) * factor, torch.sin(phase) * factor
    xa, xb = x[:, a].clone(), x[:, b].clone()
    x[:, a], x[:, b] = xa * c - xb * s, xa * s + xb * c
    return x


def turns_ref(n, base, freq_scale=1.0, ext=0.0, orig=0, factors=None, attn=1.0):
    got = []
    edge = lambda b: n * math.log(orig / (2 * math.pi * b)) / (2 * math.log(base))  # noqa: E731
    for i in range(n // 2):
        f = base ** (-2.0 * i / n) / (float(factors[i]) if factors is not None else 1.0)
        keep = 0.0
        if ext:
            lo, hi = max(0.0, math.floor(edge(32))), min(n - 1.0, math.ceil(edge(1)))
            keep = ext * (1 - min(1.0, max(0.0, (i - lo) / max(0.001, hi - lo))))
        got.append(f * (freq_scale * (1 - keep) + keep) / (2 * math.pi))
    return torch.tensor(got, dtype=torch.float64, device="cuda"), attn * (1 + 0.1 * math.log(1 / freq_scale) if ext else 1.0)


HALF_STEP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "e4m3": 2.0 ** -4}
SMALLEST = {"f16": 2.0 ** -25, "bf16": 2.0 ** -134, "e4m3": 2.0 ** -10}  # half a step of the subnormals


@pytest.mark.parametrize("typ", ["f16", "bf16", "e4m3"])
@pytest.mark.parametrize("dim,n_rot,interleaved,off", [(128, 128, False, 0), (128, 128, True, 0), (128, 64, False, 0), (64, 64, True, 0),
                                                       (64, 16, False, 0), (64, 6, False, 0), (128, 34, True, 0), (128, 2, False, 0),
                                                       (128, 128, False, 1), (64, 32, True, 3)])
def test_rope_append(be, pkg, typ, dim, n_rot, interleaved, off):
    """Ragged rows at near and far positions; `off` shifts the buffers off their 16-byte alignment."""
    torch.manual_seed(n_rot)
    lens = [(1, 1), (5, 5), (0, 0), (3, 2 ** 20 + 3), (1, 0), (2, 40), (3, 2)]
    n_kv, heads, page = 2, 6, 16
    first = [0]
    for n_q, _ in lens:
        first.append(first[-1] + n_q)
    n_tok = first[-1] + 2
    n_pages = 24
    width = -(-(2 ** 20 + 3) // page)
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    spot, free = {}, iter(torch.randperm(n_pages).tolist())
    for s, (n_q, n) in enumerate(lens):
        for j in range(max(0, n - n_q), n):
            if table[s, j // page] < 0:
                table[s, j // page] = next(free)
            spot[s, j] = (int(table[s, j // page]), j % page)
    scales = (0.0625, 0.03125) if typ == "e4m3" else (1.0, 1.0)
    k = torch.randn(n_pages, n_kv, page, dim).to(TYPES[typ]).cuda()
    v = torch.randn(n_pages, n_kv, page, dim).to(TYPES[typ]).cuda()
    k0, v0 = k.clone(), v.clone()
    cache = pkg.kv_cache(k, v, *scales)
    batch = pkg.kv_batch(table.cuda(), torch.tensor(first, dtype=torch.int32).cuda(),
                         torch.tensor([n for _, n in lens], dtype=torch.int32).cuda(), n_tok, 5)
    qd, kd = heads * dim, n_kv * dim
    buf = torch.randn(n_tok, qd + 2 * kd + off, device="cuda")[:, off:]
    q, kn, vn = buf[:, :qd], buf[:, qd:qd + kd], buf[:, qd + kd:]
    factors = (1 + torch.rand(n_rot // 2)).cuda() if interleaved else None
    rope = pkg.rope_t(n_rot, interleaved=interleaved, base=5e5, freq_factors=factors)
    table64 = be.rope_table(rope)
    turns, factor = turns_ref(n_rot, 5e5, factors=factors)
    assert torch.allclose(table64[:-1], turns, rtol=1e-13, atol=0) and float(table64[-1]) == factor
    q_out = torch.full((n_tok, qd), 9.0, device="cuda")
    be.rope_append(rope, q, kn, vn, q_out, cache, batch)
    be.synchronize()
    assert be.device_status() == 0
    touched = set()
    for s, (n_q, n) in enumerate(lens):
        for i in range(n_q):
            t, pos = first[s] + i, n - n_q + i
            if pos < 0:
                assert bool((q_out[t] == 9).all())
                continue
            # cos, sin, two products and a sum are rounded once each: 3 steps of the pair's two products
            want = rope_ref(q[t].reshape(heads, dim), pos, turns, factor, n_rot, interleaved)
            lim = 2 * q[t].abs().max().double() * 3 * 2.0 ** -24 * factor + 2 * math.pi * pos * 2.0 ** -51 * 8
            assert bool(((q_out[t].view(heads, dim).double() - want).abs() <= lim).all())
            p, at = spot[s, pos]
            touched.add((p, at))
            for pool, new, sc, turn in ((k, kn, scales[0], True), (v, vn, scales[1], False)):
                x = new[t].reshape(n_kv, dim)
                want = rope_ref(x, pos, turns, factor, n_rot, interleaved) if turn else x.double()
                got = pool[p, :, at].double() * sc
                # q's rounding, the division's, and half a step of the stored type
                lim = want.abs() * (HALF_STEP[typ] * (1 + 2.0 ** -10)) + SMALLEST[typ] * sc + 2 * x.abs().max().double() * 4 * 2.0 ** -24 + 1e-9
                assert bool(((got - want).abs() <= lim).all())
    raw = lambda x: x.view(torch.uint8)  # noqa: E731
    same_k, same_v = (raw(k) == raw(k0)).view(n_pages, n_kv, page, -1).all(-1).all(1), (raw(v) == raw(v0)).view(n_pages, n_kv, page, -1).all(-1).all(1)
    for p in range(n_pages):
        for at in range(page):
            if (p, at) not in touched:
                assert bool(same_k[p, at]) and bool(same_v[p, at])
    assert bool((q_out[first[-1]:] == 9).all())
    # in place, and each half alone
    q2 = q.clone()
    be.rope_append(rope, q2, None, None, q2, cache, batch)
    live = [first[s] + i for s, (n_q, n) in enumerate(lens) for i in range(n_q) if n - n_q + i >= 0]
    assert torch.equal(q2[live], q_out[live])
    k1 = k.clone()
    k.copy_(k0)
    v.copy_(v0)
    be.rope_append(rope, None, kn, vn, None, cache, batch)
    be.synchronize()
    assert torch.equal(raw(k), raw(k1))


@pytest.mark.parametrize("kw", [dict(freq_scale=0.25), dict(freq_scale=0.25, ext_factor=1.0, n_ctx_orig=4096),
                                dict(freq_scale=0.125, ext_factor=0.5, n_ctx_orig=32768, attn_factor=1.5)])
def test_rope_scaling(be, pkg, kw):
    rope = pkg.rope_t(128, base=1e6, **kw)
    got = be.rope_table(rope)
    turns, factor = turns_ref(128, 1e6, kw.get("freq_scale", 1.0), kw.get("ext_factor", 0.0), kw.get("n_ctx_orig", 0), attn=kw.get("attn_factor", 1.0))
    assert torch.allclose(got[:-1], turns, rtol=1e-13, atol=0)
    assert abs(float(got[-1]) / factor - 1) < 1e-7  # freq_scale and attn_factor are fp32 arguments


def test_append_saturates_and_keeps_nan(be, pkg):
    for typ, top in (("f16", 65504.0), ("e4m3", 448.0)):
        k = torch.zeros(2, 1, 16, 64).to(TYPES[typ]).cuda()
        cache = pkg.kv_cache(k, k.clone())
        batch = pkg.kv_batch(torch.zeros(1, 1, dtype=torch.int32).cuda(), torch.tensor([0, 1], dtype=torch.int32).cuda(),
                             torch.tensor([3], dtype=torch.int32).cuda(), 1, 1)
        x = torch.zeros(1, 64, device="cuda")
        x[0, :5] = torch.tensor([1e30, -1e30, float("inf"), float("-inf"), float("nan")])
        be.rope_append(None, None, x, x, None, cache, batch)
        got = cache.k[0, 0, 2].float()
        assert got[:4].tolist() == [top, -top, top, -top] and math.isnan(float(got[4])) and bool((got[5:] == 0).all())


def test_append_to_a_bad_page_stores_nothing(be, pkg):
    k = torch.full((4, 2, 16, 64), 3.0, dtype=torch.bfloat16, device="cuda")
    cache = pkg.kv_cache(k[:3], k[:3].clone())
    for bad in (-1, 3, 2 ** 31 - 1, -2 ** 31):
        batch = pkg.kv_batch(torch.tensor([[bad]], dtype=torch.int32).cuda(), torch.tensor([0, 1], dtype=torch.int32).cuda(),
                             torch.tensor([1], dtype=torch.int32).cuda(), 1, 1)
        x = torch.ones(1, 128, device="cuda")
        be.rope_append(None, None, x, x, None, cache, batch)
        be.synchronize()
        assert be.device_status() == 1 and bool((k == 3).all())


# ---- pages ----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("typ", ["bf16", "e4m3"])
@pytest.mark.parametrize("layers,n_kv,page,dim,moves", [(1, 1, 16, 64, 1), (3, 2, 32, 128, 5), (65, 1, 16, 64, 2), (2, 8, 128, 128, 7)])
def test_copy_pages(be, pkg, typ, layers, n_kv, page, dim, moves):
    torch.manual_seed(layers)
    n_pages = 2 * moves + 3
    pool = torch.randint(0, 120, (n_pages, layers, 2, n_kv, page, dim * (1 if typ == "e4m3" else 2)), dtype=torch.uint8, device="cuda").view(TYPES[typ])
    want = pool.clone()
    caches = [pkg.kv_cache(pool[:, l, 0], pool[:, l, 1]) for l in range(layers)]  # pages of the layers interleaved
    order = torch.randperm(n_pages)[:2 * moves].to(torch.int32)
    src, dst = order[:moves].cuda(), order[moves:].cuda()
    want.view(torch.uint8)[dst.long()] = want.view(torch.uint8)[src.long()]
    be.kv_copy_pages(caches, src, dst)
    be.synchronize()
    assert torch.equal(pool.view(torch.uint8), want.view(torch.uint8))
    assert be.device_status() == 0


def test_one_page_copied_to_all_others(be, pkg):
    """A sequence forked into as many as the pool holds: one source, every other page a copy."""
    pool = torch.randn(9, 2, 16, 64, device="cuda").to(torch.bfloat16)
    cache = pkg.kv_cache(pool, pool.clone())
    dst = torch.tensor([p for p in range(9) if p != 4], dtype=torch.int32).cuda()
    be.kv_copy_pages([cache], torch.full_like(dst, 4), dst)
    be.synchronize()
    assert all(torch.equal(pool[p], pool[4]) and torch.equal(cache.v[p], cache.v[4]) for p in range(9)) and be.device_status() == 0


def test_copy_pages_bad_pairs_are_left_out(be, pkg):
    pool = torch.randn(8, 2, 16, 64, device="cuda").to(torch.bfloat16)
    cache = pkg.kv_cache(pool, pool.clone())
    k0 = pool.clone()
    be.kv_copy_pages([cache], torch.tensor([0, -1, 8, 1], dtype=torch.int32).cuda(), torch.tensor([5, 6, 7, 99], dtype=torch.int32).cuda())
    be.synchronize()
    assert be.device_status() == 1
    k0[5] = k0[0]
    assert torch.equal(pool, k0)


def test_remap(be, pkg):
    torch.manual_seed(1)
    t = torch.randint(-2, 52, (7, 300), dtype=torch.int32).cuda()
    m = torch.randperm(50).to(torch.int32).cuda()
    want = torch.where((t >= 0) & (t < 50), m[t.long().clamp(0, 49)], t)
    out = torch.empty_like(t)
    be.kv_remap(t, m, out)
    assert torch.equal(out, want)
    be.kv_remap(t[:, 3:200], m)
    assert torch.equal(t[:, 3:200], want[:, 3:200]) and torch.equal(t[:, 200:] == want[:, 200:], out[:, 200:] == t[:, 200:])


# ---- together --------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("typ", ["bf16", "e4m3"])
def test_pool_prompt_fork_decode_compact(be, pkg, typ):
    """Two prompts, a fork, decode steps of all three, one leaves, the pool is compacted, more steps.  What lands in
    the cache is held to rounding and then kept densely beside it; attention is held to that book, so a page lost by
    a fork or a move shows."""
    torch.manual_seed(5)
    n_kv, group, dim, page, layers = 2, 4, 64, 16, 2
    pool = pkg.KvPool(64, page)
    mem = torch.zeros(layers, 2, 64, n_kv, page, dim, dtype=TYPES[typ], device="cuda")
    caches = [pkg.kv_cache(mem[l, 0], mem[l, 1]) for l in range(layers)]
    rope = pkg.rope_t(dim, base=1e4)
    be.rope_table(rope)
    turns, factor = turns_ref(dim, 1e4)
    book = {}  # sequence -> per layer (k, v) as stored
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731

    def step(sids, new):
        moves = [m for s, n in zip(sids, new) for m in pool.extend(s, n)]
        if moves:
            be.kv_copy_pages(caches, i32([a for a, _ in moves]), i32([b for _, b in moves]))
        batch = pool.batch(sids, new, 20)
        scratch = pkg.alloc_attn_scratch(n_kv * group, caches[0], batch)
        for l, cache in enumerate(caches):
            qkv = torch.randn(batch.n_tok, (n_kv * group + 2 * n_kv) * dim, device="cuda")
            q, k, v = qkv.split([n_kv * group * dim, n_kv * dim, n_kv * dim], 1)
            out = torch.empty(batch.n_tok, n_kv * group * dim, device="cuda")
            call = pkg.attn_call(q, k, v, out, cache, batch, scratch, rope)
            call.validate()
            call.run(be)
            be.synchronize()
            row = 0
            for s, n in zip(sids, new):
                held = book.setdefault(s, [[[], []] for _ in range(layers)])[l]
                for i in range(n):
                    pos = pool.length(s) - n + i
                    at = pool.pages(s)[pos // page], slice(None), pos % page
                    for x, (src, turn) in enumerate(((k, True), (v, False))):
                        want = src[row].reshape(n_kv, dim).double()
                        want = rope_ref(want, pos, turns, factor, dim, False) if turn else want
                        got = (cache.k, cache.v)[x][at].double()
                        lim = want.abs() * HALF_STEP[typ] * (1 + 2.0 ** -10) + SMALLEST[typ] + src[row].abs().max().double() * 2.0 ** -21
                        assert bool(((got - want).abs() <= lim).all())
                        held[x].append(got)
                    row += 1
            row = 0
            for s, n in zip(sids, new):
                K, V = (torch.stack(x, 1).repeat_interleave(group, 0) for x in book[s][l])
                for i in range(n):
                    m = pool.length(s) - n + i + 1
                    xk = q[row].double().view(-1, 1, dim) * K[:, :m]
                    w = torch.softmax(xk.sum(-1) / math.sqrt(dim), -1)
                    want = torch.einsum("hj,hjd->hd", w, V[:, :m]).flatten()
                    a = float(xk.abs().sum(-1).max()) / math.sqrt(dim)
                    split = split_error(TYPES[typ], group * batch.max_q)
                    lim = float(V[:, :m].abs().max()) * (2 * a * (split + (dim + 8) * 2.0 ** -24) + split + 2.0 ** -21 + 2 * (m / 16 + 32) * 2.0 ** -24)
                    assert bool(((out[row].double() - want).abs() <= lim).all())
                    row += 1
        assert be.device_status() == 0

    a, b = pool.new(), pool.new()
    step([a, b], [37, 50])
    c = pool.fork(a)
    book[c] = [[list(x) for x in layer] for layer in book[a]]
    for _ in range(3):
        step([a, b, c], [1, 1, 1])
    pool.free(b)
    moves, new = pool.compact()
    assert moves
    be.kv_copy_pages(caches, i32([x for x, _ in moves]), i32([y for _, y in moves]))
    for _ in range(14):
        step([c, a], [1, 1])
    step([a, c], [20, 3])


@pytest.mark.parametrize("TB", [1, 3])
def test_layer_with_attention_in_a_graph(be, pkg, TB):
    """A dense layer with its attention, step by step through a recorded plan: each step's o call sees the attention
    over the cache as the steps before left it.  The plan's calls one by one give the same bits."""
    from sycl_infer_b200.backend import alloc_act, gemv_seg
    from sycl_infer_b200.plan import SegPlan
    torch.manual_seed(2)
    hidden, heads, n_kv, dim, page = 256, 4, 2, 64, 16
    qd, kd = heads * dim, n_kv * dim
    Q4 = pkg.synth.Q4_K
    w = {n: torch.from_numpy(pkg.synth.make_weight(Q4, r, c, i)).cuda() for i, (n, r, c) in
         enumerate([("q", qd, hidden), ("k", kd, hidden), ("v", kd, hidden), ("o", hidden, qd)])}
    mem = torch.zeros(2, 2, 8 * TB, n_kv, page, dim, dtype=torch.bfloat16, device="cuda")
    caches = [pkg.kv_cache(mem[i, 0], mem[i, 1]) for i in range(2)]
    pool = pkg.KvPool(8 * TB, page)
    sids = [pool.new() for _ in range(TB)]
    for s in sids:
        pool.extend(s, 1)
    batch = pool.batch(sids, [1] * TB, 6)
    rope = pkg.rope_t(dim, base=1e4)
    be.rope_table(rope)
    scratch = pkg.alloc_attn_scratch(heads, caches[0], batch)
    x = torch.randn(TB, hidden, device="cuda")
    outs, plans = [], []
    for cache in caches:
        qkv, att, out = (torch.zeros(TB, n, device="cuda") for n in (qd + 2 * kd, qd, hidden))
        act, act_o = alloc_act(TB, hidden), alloc_act(TB, qd)
        seg = lambda n, K, rows, o, stride, col, act: gemv_seg(w=w[n], type=Q4, K=K, n_rows=rows, out=o.view(-1)[col:], out_stride=stride, alpha=0.02, x8=act[0], xmeta=act[1], xsumq=act[2])  # noqa: E731
        plan = SegPlan()
        plan.begin_call(TB)
        for n, rows, col in (("q", qd, 0), ("k", kd, qd), ("v", kd, qd + kd)):
            plan.add(seg(n, hidden, rows, qkv, qd + 2 * kd, col, act))
        plan.set_xq(x)
        q, k, v = qkv.split([qd, kd, kd], 1)
        plan.begin_attn_call(pkg.attn_call(q, k, v, att, cache, batch, scratch, rope))
        plan.begin_call(TB)
        plan.add(seg("o", qd, hidden, out, hidden, 0, act_o))
        plan.set_xq(att)
        plan.finalize()
        outs.append((out, att))
        plans.append(plan)
    stream = torch.cuda.Stream()
    plans[0].record(be, stream)
    for n in range(1, 40):
        if n > 1:
            for s in sids:
                pool.extend(s, 1)
        now = pool.batch(sids, [1] * TB, 6)
        batch.kv_len.copy_(now.kv_len)
        batch.page_table.copy_(now.page_table)
        x.normal_()
        torch.cuda.synchronize()
        plans[0].replay()
        torch.cuda.synchronize()
        plans[1].run(be)
        be.synchronize()
        assert torch.equal(outs[0][1], outs[1][1]) and torch.equal(outs[0][0], outs[1][0])
        assert float(outs[0][1].abs().max()) > 0
    assert torch.equal(mem[0], mem[1]) and be.device_status() == 0
    assert plans[0].launches() == (4 if TB == 1 else 6)


def test_dense_layer_attaches_attention(be, pkg):
    from sycl_infer_b200.layer import DenseLayer
    lay = DenseLayer(be, hidden=256, n_head=4, n_kv=2, head_dim=64, n_ff=512)
    mem = torch.zeros(2, 4, 2, 16, 64, dtype=torch.float16, device="cuda")
    cache = pkg.kv_cache(mem[0], mem[1])
    pool = pkg.KvPool(4, 16)
    s = pool.new()
    pool.extend(s, 1)
    batch = pool.batch([s], [1], 4)
    before = lay.launches_per_step()
    lay.attach_attention(cache, batch, pkg.alloc_attn_scratch(4, cache, batch))
    assert lay.launches_per_step() == before + 2
    x, out = torch.randn(1, 256, device="cuda"), torch.empty(1, 256, device="cuda")
    lay.forward(x, out)
    be.synchronize()
    # the first token attends to itself alone: its v in fp16, for every head of the group
    want = lay.qkv[0, -128:].half().float().view(2, 1, 64).expand(2, 2, 64).reshape(-1)
    assert torch.allclose(lay.attn[0], want, rtol=2.0 ** -20, atol=0)
    with pytest.raises(ValueError):
        lay.attach_attention(cache, pool.batch([s, s], [1, 1], 4), None)
