"""Workloads of the attention-side operators, and the same operators in elementary torch operations.

Four operators of a decoder layer that stand between the q|k|v call and the o call: rotary positions
with the append of K and V to a paged cache, attention over that cache for one new token (or a few) of
each sequence, the same for the many tokens of a prompt, and the copies that fork and compact a cache.
`run` computes them plainly (32-bit torch operations, 64 bits for the rotary angles) or, with `own`
set, through the library.  Sequence lengths follow from the case alone; the values from the seed.
"""
import math
import random

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
LARGEST = {"f16": 65504.0, "bf16": 3.3895313892515355e38, "e4m3": 448.0}
SCALES = {"f16": (1.0, 1.0), "bf16": (1.0, 1.0), "e4m3": (0.0625, 0.03125)}  # an 8-bit cache is scaled to its range
DENSE = {"heads": 40, "kv": 8, "dim": 128}  # the dense layer that bench.py names


def _append(name, **kw):
    d = {"name": name, "op": "append", **DENSE, "page": 32, "type": "bf16", "n_seq": 1, "q_lo": 1, "q_hi": 1, "past_lo": 0,
         "past_hi": 0, "idle": 0, "spare": 0, "mix": 1, "n_rot": 128, "interleaved": False, "base": 1e6, "freq_scale": 1.0,
         "ext": 0.0, "orig": 0, "factors": False}
    return {**d, **kw}


def _attn(name, **kw):
    d = {"name": name, "op": "attn", **DENSE, "page": 32, "type": "bf16", "n_seq": 1, "q_lo": 1, "q_hi": 1, "past_lo": 0,
         "past_hi": 0, "idle": 0, "spare": 0, "mix": 1, "window": 0, "sinks": 0}
    return {**d, **kw}


def _pages(name, **kw):
    d = {"name": name, "op": "pages", "layers": 32, "kv": 8, "dim": 128, "page": 32, "type": "bf16", "pages": 128, "moves": 1,
         "n_seq": 1, "width": 8, "remap": False}
    return {**d, **kw}


def listed():
    return [
        # one user's next token: all latency
        _append("append, 1 token", past_lo=4998, past_hi=4998),
        # a prompt's second chunk in a context stretched four times
        _append("append, 2048 tokens, yarn", q_lo=2048, q_hi=2048, past_lo=6144, past_hi=6144, type="f16", page=64,
                freq_scale=0.25, ext=1.0, orig=32768, base=1e6),
        # chunks of many requests in one step, half of the head rotated, far positions, 8-bit cache
        _append("append, ragged, part of the head", n_seq=48, q_lo=1, q_hi=37, past_lo=0, past_hi=900001, idle=2, spare=5,
                heads=32, kv=4, n_rot=64, interleaved=True, type="e4m3", page=16, base=5e5, factors=True, mix=7),
        # one user early in a chat: all latency
        _attn("decode, 1 x 517", past_lo=516, past_hi=516),
        # one user over a book: one long axis, little else to split
        _attn("decode, 1 x 131071", past_lo=131070, past_hi=131070),
        # a server's step over requests of mixed age
        _attn("decode, 32 x to 8192", n_seq=32, past_lo=200, past_hi=8191, type="f16", page=64, idle=1, spare=3, mix=3),
        # a full server with a sliding window, 8-bit cache, and drafts of one to three tokens to verify
        _attn("decode, 192 x window 1024", n_seq=192, q_lo=1, q_hi=3, past_lo=100, past_hi=6000, type="e4m3", page=16,
              heads=32, kv=8, dim=64, window=1024, sinks=4, mix=4),
        # a prompt from its first token
        _attn("prompt, 2048", q_lo=2048, q_hi=2048),
        # the last chunk of a long document
        _attn("prompt, 512 after 32001", q_lo=512, q_hi=512, past_lo=32001, past_hi=32001, type="f16", page=64),
        # prompts of odd lengths side by side, sliding window with sinks, 8-bit cache
        _attn("prompt, 7 ragged, window 512", n_seq=7, q_lo=33, q_hi=1500, past_lo=0, past_hi=2500, type="e4m3", page=16,
              heads=32, kv=8, dim=64, window=512, sinks=4, spare=9, mix=5),
        # a request forked into four answers: the last page of each is copied in every layer
        _pages("fork, 3 pages x 32 layers", moves=3, pages=64),
        # a pool tidied after many requests have left
        _pages("compact, 301 pages x 24 layers", layers=24, moves=301, pages=700, type="e4m3", page=64, n_seq=200,
               width=257, remap=True),
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    kind = rng.choice(["append", "decode", "decode", "prompt", "prompt", "pages"])
    typ, page = rng.choice(list(TYPES)), rng.choice([16, 32, 64, 128])
    dim = rng.choice([64, 128])
    kv = rng.choice([1, 2, 4, 5, 8])
    group = rng.choice([1, 2, 3, 4, 5, 6, 7, 8])
    if kind == "pages":
        layers = _spread(rng, 1, 64)
        moves = _spread(rng, 1, max(1, 9000 // layers))
        c = _pages("", layers=layers, kv=kv, dim=dim, page=page, type=typ, moves=moves, pages=2 * moves + rng.randint(1, 40),
                   n_seq=_spread(rng, 1, 200), width=_spread(rng, 1, 400), remap=rng.random() < 0.5)
        while _page_bytes(c) * c["pages"] * layers > 600e6:
            c["moves"] = max(1, c["moves"] // 2)
            c["pages"] = 2 * c["moves"] + 3
            if c["moves"] == 1:
                c["layers"] = layers = max(1, layers // 2)
    elif kind == "append":
        n_seq = _spread(rng, 1, 96)
        q_hi = _spread(rng, 1, max(1, 4096 // n_seq))
        c = _append("", heads=kv * group, kv=kv, dim=dim, page=page, type=typ, n_seq=n_seq, q_lo=rng.randint(1, q_hi), q_hi=q_hi,
                    past_lo=0, past_hi=_spread(rng, 1, 1000000), idle=rng.choice([0, 0, 1]) if n_seq > 1 else 0,
                    spare=rng.choice([0, 0, 3]), mix=rng.randrange(1 << 30), n_rot=rng.choice([dim, dim, dim // 2, dim // 4]),
                    interleaved=rng.random() < 0.5, base=rng.choice([1e4, 5e5, 1e6]), factors=rng.random() < 0.3)
        if rng.random() < 0.4:
            c.update(freq_scale=rng.choice([0.5, 0.25, 0.125]), ext=rng.choice([0.0, 1.0]), orig=rng.choice([4096, 32768]))
    else:
        window = rng.choice([0, 0, _spread(rng, 1, 5000)])
        c = _attn("", heads=kv * group, kv=kv, dim=dim, page=page, type=typ, mix=rng.randrange(1 << 30), window=window,
                  sinks=rng.choice([0, 1, 4, 130]) if window else 0, spare=rng.choice([0, 0, 2]))
        if kind == "decode":
            n_seq = _spread(rng, 1, 200)
            c.update(n_seq=n_seq, q_hi=rng.choice([1, 1, 1, 2, 4]), past_hi=_spread(rng, 1, 131072 // n_seq),
                     idle=rng.choice([0, 0, 1]) if n_seq > 1 else 0)
        else:
            n_seq = _spread(rng, 1, 8)
            q_hi = _spread(rng, 40, 2048 // n_seq)
            c.update(n_seq=n_seq, q_lo=rng.randint(1, q_hi), q_hi=q_hi, past_hi=_spread(rng, 1, 16000 // n_seq))
            while work(c)["flops"] > 300e9:
                c["past_hi"] = c["past_hi"] // 2
    del c["name"]
    return c


def _lengths(case):
    """(new tokens, length of the cache with them) of each sequence."""
    rng = random.Random(case["mix"])
    got = []
    for s in range(case["n_seq"]):
        if s < case["idle"]:
            got.append((1, 0))  # a slot of the batch that holds no sequence: its row sees nothing
            continue
        q = rng.randint(case["q_lo"], case["q_hi"])
        got.append((q, q + rng.randint(case["past_lo"], case["past_hi"])))
    return got


def _page_bytes(case):
    return case["kv"] * case["page"] * case["dim"] * (1 if case["type"] == "e4m3" else 2)


def _values(shape, typ, gen, scale=1.0):
    """Normal values in the cache's type, a slice at a time."""
    t = torch.empty(shape, dtype=TYPES[typ], device="cuda")
    flat = t.view(-1)
    step = 1 << 27
    for i in range(0, flat.numel(), step):
        n = min(step, flat.numel() - i)
        flat[i:i + n] = (torch.randn(n, generator=gen, device="cuda") / scale).to(TYPES[typ])
    return t


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    state = {"case": case}
    ks, vs = SCALES[case["type"]]
    if case["op"] == "pages":
        shape = (case["layers"], case["pages"], case["kv"], case["page"], case["dim"])
        state["k"], state["v"] = _values(shape, case["type"], gen), _values(shape, case["type"], gen)
        order = torch.randperm(case["pages"], generator=gen, device="cuda").to(torch.int32)
        state["src"], state["dst"] = order[:case["moves"]].clone(), order[case["moves"]:2 * case["moves"]].clone()
        if case["remap"]:
            state["table"] = torch.randint(-1, case["pages"], (case["n_seq"], case["width"]), generator=gen, device="cuda",
                                           dtype=torch.int32)
            state["map"] = torch.arange(case["pages"], device="cuda", dtype=torch.int32)
            state["map"][state["src"].long()] = state["dst"]
            state["new_table"] = torch.empty_like(state["table"])
    else:
        lens = _lengths(case)
        first = [0]
        for q, _ in lens:
            first.append(first[-1] + q)
        n_tok, max_q = first[-1] + case["spare"], max(q for q, _ in lens)
        held = []  # pages of each sequence that hold something: append's are those that it writes
        for q, n in lens:
            lo = (n - q) // case["page"] if case["op"] == "append" and n else 0
            used = set(range(lo, -(-n // case["page"])))
            if case["op"] == "attn" and case["window"]:  # what no new token sees any more is back in the pool
                oldest = max(0, n - q - case["window"] + 1)
                used = {p for p in used if (p + 1) * case["page"] > oldest or p * case["page"] < case["sinks"]}
            held.append(sorted(used))
        n_pages = sum(len(p) for p in held) + 3
        order = torch.randperm(n_pages - 1, generator=gen, device="cuda").to(torch.int32).cpu()
        width = max(1, max(-(-n // case["page"]) for _, n in lens))
        table, at = torch.full((case["n_seq"], width), -1, dtype=torch.int32), 0
        for s, p in enumerate(held):
            table[s, torch.tensor(p, dtype=torch.long)] = order[at:at + len(p)]
            at += len(p)
        state["table"] = table.cuda()
        state["q_start"] = torch.tensor(first, dtype=torch.int32, device="cuda")
        state["kv_len"] = torch.tensor([n for _, n in lens], dtype=torch.int32, device="cuda")
        state["max_q"] = max_q
        shape = (n_pages, case["kv"], case["page"], case["dim"])
        state["k"], state["v"] = _values(shape, case["type"], gen, ks), _values(shape, case["type"], gen, vs)
        qd, kd = case["heads"] * case["dim"], case["kv"] * case["dim"]
        # the q|k|v call's output: one row a token, the three side by side
        qkv = torch.randn(n_tok, qd + 2 * kd, generator=gen, device="cuda")
        state["q"], state["k_new"], state["v_new"] = qkv[:, :qd], qkv[:, qd:qd + kd], qkv[:, qd + kd:]
        state["out"] = torch.randn(n_tok, qd, generator=gen, device="cuda")
        if case["op"] == "append":
            state["factors"] = 1.0 + 7.0 * torch.rand(case["n_rot"] // 2, generator=gen, device="cuda") if case["factors"] else None
            state["turns"] = _turns(case, state["factors"])
    if own:
        _handles(state)
    return state


def _handles(state):
    """What a user's program keeps from step to step: the backend, the cache's and the batch's
    descriptions, the rotary table, the workspace."""
    import __graft_entry__ as entry
    pkg = entry.load_package()
    case = state["case"]
    ks, vs = SCALES[case["type"]]
    state["be"] = be = pkg.make_cuda_backend(0)
    if case["op"] == "pages":
        state["cache"] = [pkg.kv_cache(k, v) for k, v in zip(state["k"], state["v"])]
        return
    state["cache"] = pkg.kv_cache(state["k"], state["v"], k_scale=ks, v_scale=vs)
    state["batch"] = pkg.kv_batch(state["table"], state["q_start"], state["kv_len"], state["q"].shape[0], state["max_q"])
    if case["op"] == "append":
        state["rope"] = pkg.rope_t(n_rot=case["n_rot"], interleaved=case["interleaved"], base=case["base"],
                                   freq_scale=case["freq_scale"], ext_factor=case["ext"], n_ctx_orig=case["orig"],
                                   freq_factors=state["factors"])
        be.rope_table(state["rope"])
    else:
        state["scratch"] = pkg.alloc_attn_scratch(case["heads"], state["cache"], state["batch"])


# ---- the operators, plainly --------------------------------------------------------------------------

def _tokens(state):
    """Of each row: its sequence, its place among the sequence's new tokens, its position, and whether it is one."""
    rows = torch.arange(state["q"].shape[0], device="cuda")
    first = state["q_start"].long()
    seq = torch.searchsorted(first[1:], rows, right=True).clamp(max=first.numel() - 2)
    i = rows - first[seq]
    pos = state["kv_len"].long()[seq] - (first[seq + 1] - first[seq]) + i
    return seq, i, pos, rows < first[-1]


def _turns(case, factors):
    """Turns a position, in 64 bits, of each rotated pair, and the factor on the rotated values."""
    n = case["n_rot"]
    i = torch.arange(n // 2, device="cuda", dtype=torch.float64)
    theta = case["base"] ** (-2.0 * i / n)
    if factors is not None:
        theta = theta / factors.double()
    if not case["ext"]:
        return theta * case["freq_scale"] / (2 * math.pi), 1.0
    low, high = (n * math.log(case["orig"] / (beta * 2 * math.pi)) / (2 * math.log(case["base"])) for beta in (32.0, 1.0))
    low, high = max(0.0, math.floor(low)), min(n - 1.0, math.ceil(high))
    keep = (1.0 - ((i - low) / max(0.001, high - low)).clamp(0, 1)) * case["ext"]
    return (theta * case["freq_scale"] * (1 - keep) + theta * keep) / (2 * math.pi), 1.0 + 0.1 * math.log(1.0 / case["freq_scale"])


def _rotate(x, cos, sin, n, interleaved):
    a, b = (x[..., 0:n:2], x[..., 1:n:2]) if interleaved else (x[..., :n // 2], x[..., n // 2:n])
    ra, rb = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((ra, rb), -1).flatten(-2) if interleaved else torch.cat((ra, rb), -1)
    return torch.cat((turned, x[..., n:]), -1)


def _append_plain(state):
    case, k, v = state["case"], state["k"], state["v"]
    ks, vs = SCALES[case["type"]]
    top = LARGEST[case["type"]]
    seq, _, pos, used = _tokens(state)
    turns, mscale = state["turns"]
    angle = pos.double()[:, None] * turns
    angle = (angle - angle.round()) * (2 * math.pi)
    cos, sin = ((f(angle) * mscale).float()[:, None] for f in (torch.cos, torch.sin))
    n_tok, dim = pos.numel(), case["dim"]
    q = _rotate(state["q"].reshape(n_tok, case["heads"], dim), cos, sin, case["n_rot"], case["interleaved"])
    used = used & (pos >= 0)
    state["out"].copy_(torch.where(used[:, None], q.reshape(n_tok, -1), state["out"]))
    k_new = _rotate(state["k_new"].reshape(n_tok, case["kv"], dim), cos, sin, case["n_rot"], case["interleaved"]) / ks
    v_new = state["v_new"].reshape(n_tok, case["kv"], dim) / vs
    at = pos.clamp(min=0)
    page = torch.where(used, state["table"].long()[seq, at // case["page"]], k.shape[0])
    for pool, new in ((k, k_new), (v, v_new)):  # what has no place writes the last page, which holds nothing, back
        if pool.dtype == torch.float8_e4m3fn:
            pool = pool.view(torch.uint8)
            new = new.clamp(-top, top).to(torch.float8_e4m3fn).view(torch.uint8)
        else:
            new = new.clamp(-top, top).to(pool.dtype)
        flat = pool.permute(0, 2, 1, 3)
        slot = (page * case["page"] + at % case["page"]).clamp(max=k.shape[0] * case["page"] - 1)
        old = flat[slot // case["page"], slot % case["page"]]
        keep = (page < k.shape[0])[:, None, None]
        flat[slot // case["page"], slot % case["page"]] = torch.where(keep, new, old)
    return {"q": state["out"], "k": k, "v": v}


def _attn_plain(state):
    case = state["case"]
    ks, vs = SCALES[case["type"]]
    n_seq, kv, dim, group = case["n_seq"], case["kv"], case["dim"], case["heads"] // case["kv"]
    first, lens, max_q = state["q_start"].long(), state["kv_len"].long(), state["max_q"]
    n_q = first[1:] - first[:-1]
    table = state["table"].long()
    width = table.shape[1] * case["page"]

    def gathered(pool, scale):
        x = pool.view(torch.uint8) if pool.dtype == torch.float8_e4m3fn else pool
        x = x[table.clamp(min=0)].view(pool.dtype).float() * scale  # [n_seq, pages, kv, page, dim]
        return x.permute(0, 2, 1, 3, 4).reshape(n_seq, kv, width, dim)

    i = torch.arange(max_q, device="cuda")
    row = (first[:-1, None] + i).clamp(max=state["q"].shape[0] - 1)
    q = state["q"].reshape(-1, kv, group, dim)[row]  # [n_seq, max_q, kv, group, dim]
    q = q.permute(0, 2, 3, 1, 4).reshape(n_seq, kv, group * max_q, dim)
    score = torch.matmul(q, gathered(state["k"], ks).transpose(-1, -2)).mul_(dim ** -0.5)
    pos = (lens - n_q)[:, None] + i
    j = torch.arange(width, device="cuda")
    seen = (j <= pos[:, :, None]) & (table >= 0).repeat_interleave(case["page"], 1)[:, None]
    if case["window"]:
        seen &= (j > pos[:, :, None] - case["window"]) | (j < case["sinks"])
    score = score.view(n_seq, kv, group, max_q, width).masked_fill_(~seen[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(n_seq, kv, group * max_q, width), gathered(state["v"], vs)).view(n_seq, kv, group, max_q, dim)
    out = torch.where(total > 0, out / total, 0.0).permute(0, 3, 1, 2, 4).reshape(n_seq, max_q, -1)
    seq, at, _, used = _tokens(state)
    state["out"].copy_(torch.where(used[:, None], out[seq, at.clamp(0, max_q - 1)], state["out"]))
    return state["out"]


def _pages_plain(state):
    got = {"k": state["k"], "v": state["v"]}
    src, dst = state["src"].long(), state["dst"].long()
    for pool in (state["k"], state["v"]):
        raw = pool.view(torch.uint8) if pool.dtype == torch.float8_e4m3fn else pool
        raw[:, dst] = raw[:, src]
    if state["case"]["remap"]:
        table = state["table"].long()
        state["new_table"].copy_(torch.where(table >= 0, state["map"].long()[table.clamp(min=0)], table))
        got["table"] = state["new_table"]
    return got


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"append": _append_plain, "attn": _attn_plain, "pages": _pages_plain}[op](state)
    case, be = state["case"], state["be"]
    if op == "append":
        be.rope_append(state["rope"], state["q"], state["k_new"], state["v_new"], state["out"], state["cache"], state["batch"])
        return {"q": state["out"], "k": state["k"], "v": state["v"]}
    if op == "attn":
        be.attn(state["q"], state["out"], state["cache"], state["batch"], state["scratch"], window=case["window"], n_sink=case["sinks"])
        return state["out"]
    be.kv_copy_pages(state["cache"], state["src"], state["dst"])
    if case["remap"]:
        be.kv_remap(state["table"], state["map"], state["new_table"])
        return {"k": state["k"], "v": state["v"], "table": state["new_table"]}
    return {"k": state["k"], "v": state["v"]}


# ---- what the operators are, in 64 bits and a sequence at a time ------------------------------------------

def _exact_append(state):
    case = state["case"]
    ks, vs = SCALES[case["type"]]
    n, dim, heads, kv = case["n_rot"], case["dim"], case["heads"], case["kv"]
    inv = []
    for i in range(n // 2):
        f = case["base"] ** (-2.0 * i / n)
        inv.append(f / float(state["factors"][i]) if case["factors"] else f)
    gain = 1.0
    if case["ext"]:
        edge = [n * math.log(case["orig"] / (b * 2 * math.pi)) / (2 * math.log(case["base"])) for b in (32.0, 1.0)]
        lo, hi = max(0, math.floor(edge[0])), min(n - 1, math.ceil(edge[1]))
        for i in range(n // 2):
            share = case["ext"] * (1 - min(1.0, max(0.0, (i - lo) / max(0.001, hi - lo))))
            inv[i] = inv[i] * (share + case["freq_scale"] * (1 - share))
        gain = 1 + 0.1 * math.log(1 / case["freq_scale"])
    else:
        inv = [f * case["freq_scale"] for f in inv]
    inv = torch.tensor(inv, dtype=torch.float64, device="cuda")
    pair = torch.arange(n // 2, device="cuda")
    one, two = (2 * pair, 2 * pair + 1) if case["interleaved"] else (pair, pair + n // 2)
    q_out, k_out, v_out = state["out"].double(), state["k"].double(), state["v"].double()
    start = 0
    for s, (q_len, length) in enumerate(_lengths(case)):
        rows = slice(start, start + q_len)
        start += q_len
        if length < q_len:
            continue
        pos = torch.arange(length - q_len, length, device="cuda")
        wave = torch.polar(torch.full((q_len, n // 2), gain, dtype=torch.float64, device="cuda"),
                           torch.remainder(pos.double()[:, None] * inv, 2 * math.pi))[:, None]

        def turn(x):
            x = x.double().clone()
            z = torch.complex(x[..., one], x[..., two]) * wave
            x[..., one], x[..., two] = z.real, z.imag
            return x

        q_out[rows] = turn(state["q"][rows].reshape(q_len, heads, dim)).reshape(q_len, -1)
        page = state["table"][s].long()[pos // case["page"]]
        k_out[page, :, pos % case["page"]] = turn(state["k_new"][rows].reshape(q_len, kv, dim)) / ks
        v_out[page, :, pos % case["page"]] = state["v_new"][rows].reshape(q_len, kv, dim).double() / vs
    return {"q": q_out, "k": k_out, "v": v_out}


def _exact_attn(state):
    case = state["case"]
    ks, vs = SCALES[case["type"]]
    dim, heads, group, page = case["dim"], case["heads"], case["heads"] // case["kv"], case["page"]
    out = state["out"].double()
    start = 0
    for s, (q_len, length) in enumerate(_lengths(case)):
        q = state["q"][start:start + q_len].double().view(q_len, heads, dim)
        rows = out[start:start + q_len].view(q_len, heads, dim)
        start += q_len
        oldest = max(0, length - q_len - case["window"] + 1) if case["window"] else 0
        keys = torch.arange(length, device="cuda")
        keys = keys[(keys >= oldest) | (keys < case["sinks"])]
        if not keys.numel():
            rows.zero_()
            continue
        pages = state["table"][s].long()[keys // page]
        at = torch.arange(length - q_len, length, device="cuda")[:, None]
        hidden = keys > at
        if case["window"]:
            hidden |= (keys <= at - case["window"]) & (keys >= case["sinks"])
        for h in range(case["kv"]):
            k, v = (pool[:, h][pages, keys % page].double() * c for pool, c in ((state["k"].half() if case["type"] == "e4m3" else state["k"], ks),
                                                                              (state["v"].half() if case["type"] == "e4m3" else state["v"], vs)))
            for g in range(h * group, (h + 1) * group):
                w = torch.softmax((q[:, g] @ k.T / math.sqrt(dim)).masked_fill(hidden, float("-inf")), -1)
                rows[:, g] = torch.nan_to_num(w) @ v
    return out


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(state)
    if case["op"] == "attn":
        return _exact_attn(state)
    got = {}
    for name in ("k", "v"):
        pool = state[name].half() if case["type"] == "e4m3" else state[name]
        got[name] = pool.clone()
        for a, b in zip(state["src"].tolist(), state["dst"].tolist()):
            got[name][:, b] = pool[:, a]
        got[name] = got[name].to(state[name].dtype)
    if case["remap"]:
        new = state["map"].tolist()
        rows = [[new[p] if p >= 0 else p for p in r] for r in state["table"].tolist()]
        got["table"] = torch.tensor(rows, dtype=torch.int32)
    return got


def work(case):
    if case["op"] == "pages":
        tables = 2 * 4 * case["n_seq"] * case["width"] + 4 * case["pages"] if case["remap"] else 0
        return {"bytes": 4 * case["layers"] * case["moves"] * _page_bytes(case) + 8 * case["moves"] + tables, "flops": 0}
    lens = _lengths(case)
    size = 1 if case["type"] == "e4m3" else 2
    tokens = sum(q for q, _ in lens)
    if case["op"] == "append":
        moved = tokens * case["dim"] * (8 * case["heads"] + (8 + 2 * size) * case["kv"])
        return {"bytes": moved, "flops": 3 * tokens * case["n_rot"] * (case["heads"] + case["kv"])}
    pairs = keys = 0
    for q, n in lens:
        if not case["window"]:
            keys += n
            pairs += max(0, q * n - q * (q - 1) // 2) if n >= q else 0
            continue
        keys += len(set(range(max(0, n - q - case["window"] + 1), n)) | set(range(min(n, case["sinks"]))))
        for p in range(max(0, n - q), n):
            near = min(p + 1, case["window"])
            pairs += near + min(case["sinks"], p + 1 - near)
    return {"bytes": 2 * keys * case["kv"] * case["dim"] * size + 8 * tokens * case["heads"] * case["dim"],
            "flops": 4 * pairs * case["heads"] * case["dim"]}
