"""What the paged cache's serving operators are measured on.

Three kinds of case:

  chunk   attention of a ragged batch of new tokens over a paged f16 cache, causal, optionally with a sliding
          window and a few first tokens (sinks) that stay visible; one new token per sequence is its decode form
  mrope   rotary positions with three axes (time, height, width) for a ragged batch of new tokens, whose K/V rows
          go to the pages of an f16 or an 8-bit cache
  move    pages of every layer copied at once: forks of sequences and compaction of the pool

`own` says whether `run` calls this repository's kernels or computes the plain form.
"""
import importlib
import math
import random

import torch

own = False
_foundry = None


def _library():
    package = importlib.import_module("test-burn_b200")
    global _foundry
    if _foundry is None:
        _foundry = package.Foundry(0, torch.cuda.current_stream().cuda_stream)
    return package, _foundry


# ------------------------------------------------------------------------------------------------ cases ---

def listed():
    return [
        # a speculative-decoding step: five drafted tokens of each of eight sequences are verified at once; latency counts
        dict(name="verify_8x5", kind="chunk", hq=16, hkv=2, d=128, page=16, decode=0, chunks=8, q_lo=5, q_hi=5,
             kv_lo=512, kv_hi=4096, window=0, sinks=0, freed=False, lens=1),
        # a serving step that mixes two prompt chunks with 46 sequences that decode
        dict(name="serve_mixed", kind="chunk", hq=32, hkv=8, d=128, page=16, decode=46, chunks=2, q_lo=384, q_hi=512,
             kv_lo=512, kv_hi=8192, window=0, sinks=0, freed=False, lens=2),
        # chunked prefill of two long prompts: matrix products bound it
        dict(name="prompt_chunks", kind="chunk", hq=16, hkv=2, d=128, page=64, decode=0, chunks=2, q_lo=3001, q_hi=4096,
             kv_lo=6000, kv_hi=8192, window=0, sinks=0, freed=False, lens=3),
        # one user, one token, a windowed layer: the smallest call
        dict(name="window_decode_1", kind="chunk", hq=16, hkv=2, d=128, page=16, decode=1, chunks=0, q_lo=1, q_hi=1,
             kv_lo=16000, kv_hi=16384, window=1024, sinks=4, freed=True, lens=4),
        # batched decode of a windowed layer, pages behind the window given back to the pool
        dict(name="window_decode_64", kind="chunk", hq=16, hkv=2, d=128, page=16, decode=64, chunks=0, q_lo=1, q_hi=1,
             kv_lo=512, kv_hi=16384, window=4096, sinks=4, freed=True, lens=5),
        # prompt chunks of a windowed layer with seven query heads per key head and 64-wide heads
        dict(name="window_prompt", kind="chunk", hq=14, hkv=2, d=64, page=32, decode=3, chunks=2, q_lo=1500, q_hi=4096,
             kv_lo=6000, kv_hi=12288, window=512, sinks=4, freed=False, lens=6),
        # one new token of each of 64 sequences
        dict(name="mrope_decode", kind="mrope", hq=16, hkv=2, d=128, page=16, bits=16, batch=64, q_lo=1, q_hi=1,
             kv_lo=512, kv_hi=4096, interleaved=False, lens=7),
        # prompts of text and images
        dict(name="mrope_prompt", kind="mrope", hq=32, hkv=8, d=128, page=16, bits=16, batch=3, q_lo=2000, q_hi=4096,
             kv_lo=4096, kv_hi=6000, interleaved=False, lens=8),
        # the same in front of the 8-bit cache, axes interleaved over the frequencies
        dict(name="mrope_prompt_8bit", kind="mrope", hq=16, hkv=2, d=128, page=16, bits=8, batch=3, q_lo=1000, q_hi=4096,
             kv_lo=4096, kv_hi=6000, interleaved=True, lens=9),
        # beam search or parallel samples: eight sequences get private copies of their last page, in all layers
        dict(name="fork_8", kind="move", hkv=2, d=128, page=16, bits=16, layers=36, pool=256, moves=8, fork=True),
        # the pool is compacted before it shrinks
        dict(name="compact_1000", kind="move", hkv=8, d=128, page=16, bits=16, layers=8, pool=2500, moves=1000, fork=False),
        # the same on the 8-bit cache (bytes and row scales)
        dict(name="compact_8bit", kind="move", hkv=2, d=128, page=32, bits=8, layers=28, pool=2000, moves=777, fork=False),
    ]


def _between(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["chunk", "chunk", "chunk", "mrope", "move"])
    lens = rng.randrange(1 << 20)
    if kind == "chunk":
        hkv, group, d = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 5, 7, 8]), rng.choice([64, 128])
        page = rng.choice([16, 32, 64])
        window = rng.choice([0, _between(rng, 1, 8192)])
        sinks = rng.choice([0, 0, 4, rng.randrange(1, 200)]) if window else 0
        form = rng.choice(["decode", "prompt", "mixed"])
        decode = 0 if form == "prompt" else _between(rng, 1, 64)
        chunks = 0 if form == "decode" else _between(rng, 1, 4)
        q_hi = _between(rng, 2, 2048) if chunks else 1
        kv_hi = _between(rng, max(q_hi + 1, rng.choice([1, 500, 2000])), 8192 if chunks else 16384)
        # no more scores than the largest listed case has
        while decode * kv_hi * hkv > 64 * 16384 * 2:
            decode //= 2
        while chunks * q_hi * kv_hi * hkv * group > 2 * 4096 * 8192 * 16 // 2:
            q_hi = max(2, q_hi // 2)
        q_lo = max(1, q_hi // 3) if chunks else 1
        return dict(kind="chunk", hq=hkv * group, hkv=hkv, d=d, page=page, decode=decode, chunks=chunks, q_lo=q_lo,
                    q_hi=q_hi, kv_lo=max(q_hi, kv_hi // 5), kv_hi=max(q_hi, kv_hi), window=window, sinks=sinks,
                    freed=bool(window) and not chunks and rng.random() < 0.5, lens=lens)
    if kind == "mrope":
        bits = rng.choice([16, 16, 8])
        hkv, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 7])
        batch, q_hi = _between(rng, 1, 64), _between(rng, 1, 4096)
        while batch * q_hi * (group + 2) * hkv > 12000 * 48:
            batch = max(1, batch // 2)
            q_hi = max(1, q_hi // 2)
        kv_hi = _between(rng, q_hi, 8192)
        return dict(kind="mrope", hq=hkv * group, hkv=hkv, d=128 if bits == 8 else rng.choice([64, 128]),
                    page=rng.choice([16, 32, 64]), bits=bits, batch=batch, q_lo=max(1, q_hi // 3), q_hi=q_hi,
                    kv_lo=max(q_hi, kv_hi // 4), kv_hi=kv_hi, interleaved=rng.random() < 0.5, lens=lens)
    bits = rng.choice([16, 8])
    hkv, page, layers = rng.choice([1, 2, 4, 8]), rng.choice([16, 32, 64]), _between(rng, 1, 48)
    moves = _between(rng, 1, 1500)
    while moves * hkv * page * layers > 1000 * 8 * 16 * 8:
        moves = max(1, moves // 2)
        layers = max(1, layers - 1)
    return dict(kind="move", hkv=hkv, d=128 if bits == 8 else rng.choice([64, 128]), page=page, bits=bits, layers=layers,
                pool=2 * moves + rng.randrange(8, 200), moves=moves, fork=rng.random() < 0.5)


def _lens(case):
    """(new tokens, keys after the append) of every sequence."""
    r = random.Random(case["lens"])
    if case["kind"] == "mrope":
        q = [_between(r, case["q_lo"], case["q_hi"]) for _ in range(case["batch"])]
    else:
        q = [1] * case["decode"] + [_between(r, case["q_lo"], case["q_hi"]) for _ in range(case["chunks"])]
        r.shuffle(q)
    kv = [max(n, _between(r, case["kv_lo"], case["kv_hi"])) for n in q]
    return q, kv


def _sections(case):
    """How the rotation's frequencies are shared out to time, height and width; interleaved, time has the most."""
    half = case["d"] // 2
    t = 3 * half // 8 if case["interleaved"] else half // 4
    h = (half - t) // 2
    return [t, h, half - t - h]


def _axes(case):
    """The axis of every frequency."""
    half, sec = case["d"] // 2, _sections(case)
    if not case["interleaved"]:
        return [a for a in range(3) for _ in range(sec[a])]
    return [j % 3 if j % 3 and j < 3 * sec[j % 3] else 0 for j in range(half)]


def _visible(case, n_q, n_kv):
    """(scores, keys that some query sees) of one sequence."""
    w, s = case["window"], case["sinks"]
    first = n_kv - n_q
    if not w:
        return n_q * first + n_q * (n_q + 1) // 2, n_kv
    scores = 0
    for p in (first + i for i in range(n_q)):
        lo = max(0, p - w + 1)
        scores += p + 1 - lo + min(s, lo)
    lo = max(0, first - w + 1)
    return scores, n_kv - lo + min(s, lo)


def work(case):
    d = case["d"]
    if case["kind"] == "chunk":
        total = [_visible(case, a, b) for a, b in zip(*_lens(case))]
        keys, scores, tokens = sum(t[1] for t in total), sum(t[0] for t in total), sum(_lens(case)[0])
        return {"bytes": 2 * keys * case["hkv"] * d * 2 + 2 * tokens * case["hq"] * d * 2, "flops": 4 * scores * case["hq"] * d}
    if case["kind"] == "mrope":
        tokens = sum(_lens(case)[0])
        row = 2 if case["bits"] == 16 else 1
        return {"bytes": tokens * d * (2 * case["hq"] * 2 + 2 * case["hkv"] * (2 + row)) + tokens * 12 +
                (tokens * case["hkv"] * 2 * 4 if case["bits"] == 8 else 0), "flops": 3 * tokens * d * (case["hq"] + case["hkv"])}
    row = d * 2 if case["bits"] == 16 else d + 4
    return {"bytes": 2 * 2 * case["moves"] * case["layers"] * case["hkv"] * case["page"] * row, "flops": 0}


# --------------------------------------------------------------------------------------------- prepare ---

def _pages(case, kv, g):
    """A page table over a shuffled pool; entries behind the last page of a sequence hold no page."""
    p = case["page"]
    need = [-(-n // p) for n in kv]
    pool = sum(need) + 7
    order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(kv), max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, pool


def _tables(rows, d):
    ang = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * \
        torch.pow(torch.tensor(1e6, dtype=torch.float64, device="cuda"),
                  -torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)[None]
    return ang.cos().half(), ang.sin().half()


def _begin(q):
    out = [0]
    for n in q:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32, device="cuda")


def _prepare_chunk(case, g):
    q_lens, kv = _lens(case)
    hq, hkv, d, p = case["hq"], case["hkv"], case["d"], case["page"]
    table, pool = _pages(case, kv, g)
    k = torch.randn((pool, hkv, p, d), generator=g, device="cuda", dtype=torch.float16)
    v = torch.randn((pool, hkv, p, d), generator=g, device="cuda", dtype=torch.float16)
    k[..., :: d // 4] *= 3.0  # a few wide channels, as trained keys have
    tokens = sum(q_lens)
    q = torch.randn((tokens, hq * d), generator=g, device="cuda", dtype=torch.float16)
    if case["freed"]:  # the pages that no later token sees have gone back to the pool
        for b, n in enumerate(kv):
            first, last = -(-case["sinks"] // p), max(0, n - case["window"]) // p
            if last > first:
                table[b, first:last] = -1
    s = dict(case=case, q_lens=q_lens, kv=kv, k=k, v=v, table=table, q=q, out=torch.empty_like(q),
             lens=torch.tensor(kv, dtype=torch.int32, device="cuda"), begin=_begin(q_lens))
    if own:  # one plan serves every layer of a step
        package, f = _library()
        s["plan"] = f.chunk_plan(q_lens, kv, n_heads=hq, n_kv_heads=hkv, head_dim=d, page_size=p, window=case["window"],
                                 sinks=case["sinks"])
        s["cache"] = package.paged_kv(k, v, table, s["lens"], n_kv_heads=hkv, page_size=p, head_dim=d)
    return s


def _prepare_mrope(case, g):
    q_lens, kv = _lens(case)
    hq, hkv, d, p = case["hq"], case["hkv"], case["d"], case["page"]
    table, pool = _pages(case, kv, g)
    tokens = sum(q_lens)
    qkv = [torch.randn((tokens, h * d), generator=g, device="cuda", dtype=torch.float16) for h in (hq, hkv, hkv)]
    # text counts on; images of 24 x 32 patches hold time and walk through height and width
    pos, r = [], random.Random(case["lens"] + 1)
    for n, total in zip(q_lens, kv):
        at, rows = total - n, []
        while len(rows) < n:
            if r.random() < 0.5:
                rows += [(at + i, at + i, at + i) for i in range(64)]
                at += 64
            else:
                rows += [(at, at + i // 32, at + i % 32) for i in range(768)]
                at += 32
        pos += rows[:n]
    positions = torch.tensor(pos, dtype=torch.int32).t().contiguous().cuda()
    cos, sin = _tables(max(kv) + 4096, d)
    s = dict(case=case, q=qkv[0], k_new=qkv[1], v_new=qkv[2], q_rot=torch.empty_like(qkv[0]), positions=positions, cos=cos,
             sin=sin, table=table, lens=torch.tensor(kv, dtype=torch.int32, device="cuda"), begin=_begin(q_lens),
             axes=_axes(case))
    if case["bits"] == 16:
        s["k"], s["v"] = (torch.randn((pool, hkv, p, d), generator=g, device="cuda", dtype=torch.float16) for _ in range(2))
    else:
        s["k"], s["v"] = (torch.randint(0, 120, (pool, hkv, p, d), generator=g, device="cuda", dtype=torch.uint8) for _ in range(2))
        s["ks"], s["vs"] = (torch.rand((pool, hkv, p), generator=g, device="cuda") * 0.01 for _ in range(2))
    if own:
        package, _ = _library()
        s["axes"] = package.mrope_axes(_sections(case), interleaved=case["interleaved"])
        s["cache"] = package.paged_kv(s["k"], s["v"], table, s["lens"], n_kv_heads=hkv, page_size=p, head_dim=d) \
            if case["bits"] == 16 else package.paged_kv8(s["k"], s["v"], s["ks"], s["vs"], table, s["lens"], n_kv_heads=hkv,
                                                         page_size=p)
    return s


def _prepare_move(case, g):
    hkv, d, p, layers, pool, n = (case[x] for x in ("hkv", "d", "page", "layers", "pool", "moves"))
    shape = (layers, pool, hkv, p, d)
    if case["bits"] == 16:
        s = dict(k=torch.randn(shape, generator=g, device="cuda", dtype=torch.float16),
                 v=torch.randn(shape, generator=g, device="cuda", dtype=torch.float16))
    else:
        s = dict(k=torch.randint(0, 120, shape, generator=g, device="cuda", dtype=torch.uint8),
                 v=torch.randint(0, 120, shape, generator=g, device="cuda", dtype=torch.uint8),
                 ks=torch.rand(shape[:4], generator=g, device="cuda"), vs=torch.rand(shape[:4], generator=g, device="cuda"))
    order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32).cpu()
    src, dst = order[:n].clone(), order[n:2 * n].clone()
    if case["fork"]:  # several children of one sequence copy the same page
        src = src[torch.arange(n) // 4 * 4]
    s |= dict(case=case, src=src, dst=dst, src_ids=src.cuda().long(), dst_ids=dst.cuda().long())
    if own:
        package, _ = _library()
        table = torch.zeros((1, 1), dtype=torch.int32, device="cuda")
        if case["bits"] == 16:
            caches = [package.paged_kv(s["k"][i], s["v"][i], table, table, n_kv_heads=hkv, page_size=p, head_dim=d)
                      for i in range(layers)]
        else:
            caches = [package.paged_kv8(s["k"][i], s["v"][i], s["ks"][i], s["vs"][i], table, table, n_kv_heads=hkv, page_size=p)
                      for i in range(layers)]
        s["layers"] = package.kv_layers(caches)
        s["src"], s["dst"] = src.numpy().view("uint32"), dst.numpy().view("uint32")  # the host's allocator has them
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return {"chunk": _prepare_chunk, "mrope": _prepare_mrope, "move": _prepare_move}[case["kind"]](case, g)


# ------------------------------------------------------------------------------------------- plain forms ---

def _plain_chunk(s):
    """Sequences of similar sizes are padded and computed together: scores, mask, softmax, product."""
    c = s["case"]
    hq, hkv, d, p = c["hq"], c["hkv"], c["d"], c["page"]
    groups = {}
    for b, n in enumerate(s["q_lens"]):
        groups.setdefault(n if n <= 16 else -b, []).append(b)
    out = s["out"]
    for seqs in groups.values():
        nq, nk = max(s["q_lens"][b] for b in seqs), max(s["kv"][b] for b in seqs)
        idx = torch.tensor(seqs, device="cuda")
        begin, lens = s["begin"][idx].long(), s["lens"][idx].long()
        cnt = s["begin"][idx + 1].long() - begin
        pages = s["table"][idx, : -(-nk // p)].long().clamp_(min=0)
        k = s["k"][pages].permute(0, 2, 1, 3, 4).reshape(len(seqs), hkv, -1, d)[:, :, :nk].float()
        v = s["v"][pages].permute(0, 2, 1, 3, 4).reshape(len(seqs), hkv, -1, d)[:, :, :nk].float()
        r = torch.arange(nq, device="cuda")
        rows = (begin[:, None] + r).clamp_(max=s["q"].shape[0] - 1)
        q = s["q"][rows].view(len(seqs), nq, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(len(seqs), hkv, -1, d).float()
        at = (lens - cnt)[:, None] + r  # positions of the queries
        key = torch.arange(nk, device="cuda")
        see = key[None, None] <= at[:, :, None]
        if c["window"]:
            see &= (at[:, :, None] - key < c["window"]) | (key < c["sinks"])
        see = see & (key < lens[:, None])[:, None]
        see = see[:, None, None].expand(-1, -1, hq // hkv, -1, -1).reshape(len(seqs), 1, -1, nk)
        score = (q @ k.transpose(2, 3)).mul_(1.0 / math.sqrt(d)).masked_fill_(~see, -math.inf)
        top = score.amax(-1, keepdim=True).clamp_(min=-1e30)
        weight = score.sub_(top).exp_()
        o = (weight @ v) / weight.sum(-1, keepdim=True).clamp_(min=1e-30)
        o = o.view(len(seqs), hkv, hq // hkv, nq, d).permute(0, 3, 1, 2, 4).reshape(len(seqs), nq, hq * d)
        real = r[None] < cnt[:, None]
        out[rows[real]] = o[real].half()
    return out


def _slots(s):
    """(page, row) of every new token's place in the pools."""
    c, begin = s["case"], s["begin"].long()
    token = torch.arange(s["q"].shape[0], device="cuda")
    seq = torch.searchsorted(begin, token, right=True) - 1
    slot = s["lens"].long()[seq] - (begin[seq + 1] - token)
    return s["table"].long()[seq, slot // c["page"]], slot % c["page"]


def _plain_mrope(s):
    c = s["case"]
    hq, hkv, d, p = c["hq"], c["hkv"], c["d"], c["page"]
    axis = torch.tensor(list(s["axes"]), device="cuda").long()
    freq = torch.arange(d // 2, device="cuda")
    row = s["positions"].long()[axis].t()  # [tokens, d/2]: the table row of every frequency
    cos, sin = s["cos"][row, freq].float()[:, None], s["sin"][row, freq].float()[:, None]

    def turn(x, heads):
        x = x.view(-1, heads, d).float()
        a, b = x[..., : d // 2], x[..., d // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).half()

    s["q_rot"].copy_(turn(s["q"], hq).view(-1, hq * d))
    page, at = _slots(s)
    k, v = turn(s["k_new"], hkv), s["v_new"].view(-1, hkv, d)
    if c["bits"] == 16:
        s["k"][page, :, at], s["v"][page, :, at] = k, v
        return {"q_rot": s["q_rot"], "k": s["k"], "v": s["v"]}

    def quantise(x):
        x = x.float()
        top = x.abs().amax(-1)
        scale = torch.where(top > 0, top / 448.0, torch.ones_like(top))
        return (x / scale[..., None]).to(torch.float8_e4m3fn).view(torch.uint8), scale

    kb, s["ks"][page, :, at] = quantise(k)
    vb, s["vs"][page, :, at] = quantise(v)
    s["k"][page, :, at] = kb
    s["v"].view(-1, hkv, p // 16, d, 16)[page, :, at // 16, :, at % 16] = vb
    return _eight_bit(s)


def _eight_bit(s):
    return {"q_rot": s["q_rot"], "k": s["k"].view(torch.float8_e4m3fn), "v": s["v"].view(torch.float8_e4m3fn), "ks": s["ks"],
            "vs": s["vs"]}


def _moved(s):
    if s["case"]["bits"] == 16:
        return {"k": s["k"].view(torch.int16), "v": s["v"].view(torch.int16)}
    return {"k": s["k"], "v": s["v"], "ks": s["ks"].view(torch.int32), "vs": s["vs"].view(torch.int32)}


def _plain_move(s):
    s["k"][:, s["dst_ids"]] = s["k"][:, s["src_ids"]]
    s["v"][:, s["dst_ids"]] = s["v"][:, s["src_ids"]]
    if s["case"]["bits"] == 8:
        s["ks"][:, s["dst_ids"]] = s["ks"][:, s["src_ids"]]
        s["vs"][:, s["dst_ids"]] = s["vs"][:, s["src_ids"]]
    return _moved(s)


def run(state):
    c = state["case"]
    if not own:
        return {"chunk": _plain_chunk, "mrope": _plain_mrope, "move": _plain_move}[c["kind"]](state)
    _, f = _library()
    if c["kind"] == "chunk":
        f.paged_chunk_attention(state["plan"], state["cache"], state["q"], state["out"])
        return state["out"]
    if c["kind"] == "mrope":
        f.paged_mrope_append(state["cache"], state["q"], state["k_new"], state["v_new"], state["q_rot"], state["cos"],
                             state["sin"], state["positions"], state["begin"], state["axes"], n_heads=c["hq"])
        return {"q_rot": state["q_rot"], "k": state["k"], "v": state["v"]} if c["bits"] == 16 else _eight_bit(state)
    f.paged_move_pages(state["layers"], state["src"], state["dst"])
    return _moved(state)


# ------------------------------------------------------------------------------------------------- exact ---

def exact(case, seed):
    """From the definitions, in 64 bits, sequence by sequence and head by head."""
    if case["kind"] == "move":
        return None  # bits that move: nothing is computed
    s = prepare(case, seed)
    hq, hkv, d, p = case["hq"], case["hkv"], case["d"], case["page"]
    q_lens, kv = _lens(case)
    if case["kind"] == "chunk":
        out = torch.zeros((sum(q_lens), hq, d), dtype=torch.float64, device="cuda")
        start = 0
        for b, (n, total) in enumerate(zip(q_lens, kv)):
            keys = torch.arange(total, device="cuda")
            page = s["table"][b].long()[keys // p].clamp(min=0)
            for h in range(hq):
                k = s["k"][page, h // (hq // hkv), keys % p].double()
                v = s["v"][page, h // (hq // hkv), keys % p].double()
                q = s["q"].view(-1, hq, d)[start:start + n, h].double()
                dist = torch.arange(total - n, total, device="cuda")[:, None] - keys[None]
                hidden = dist < 0
                if case["window"]:
                    hidden |= (dist >= case["window"]) & (keys >= case["sinks"])
                z = torch.where(hidden, -math.inf, torch.mm(q, k.t()) / math.sqrt(d))
                out[start:start + n, h] = torch.mm(torch.exp(z - torch.logsumexp(z, 1, keepdim=True)), v)
                del z, hidden, dist
            start += n
        return out.view(-1, hq * d)
    cos, sin = s["cos"].double(), s["sin"].double()
    axis = torch.tensor(_axes(case), device="cuda")

    def turned(x, heads):
        z = torch.view_as_complex(torch.stack(x.double().view(-1, heads, 2, d // 2).unbind(2), -1))
        w = torch.stack([torch.complex(cos[s["positions"][a].long()], sin[s["positions"][a].long()]) for a in range(3)])
        w = w.gather(0, axis.expand(1, w.shape[1], -1))[0]
        z = z * w[:, None]
        return torch.cat([z.real, z.imag], -1)

    q, k, v = turned(s["q"], hq), turned(s["k_new"], hkv), s["v_new"].double().view(-1, hkv, d)
    page, at = [], []
    for b, (n, total) in enumerate(zip(q_lens, kv)):
        slot = torch.arange(total - n, total, device="cuda")
        page.append(s["table"][b].long()[slot // p])
        at.append(slot % p)
    page, at = torch.cat(page), torch.cat(at)
    if case["bits"] == 16:
        kp, vp = s["k"].double(), s["v"].double()
        kp[page, :, at], vp[page, :, at] = k, v
        return {"q_rot": q.view(-1, hq * d), "k": kp, "v": vp}
    kp, vp = s["k"].view(torch.float8_e4m3fn).double(), s["v"].view(torch.float8_e4m3fn).double()
    ks, vs = s["ks"].double(), s["vs"].double()
    k = k.half().double()  # the format quantises the rotated row as the f16 cache would hold it
    ks[page, :, at], vs[page, :, at] = k.abs().amax(-1) / 448, v.abs().amax(-1) / 448
    kp[page, :, at] = k / (k.abs().amax(-1, keepdim=True) / 448)
    dims = vp.view(-1, hkv, p // 16, d, 16)
    dims[page, :, at // 16, :, at % 16] = v / (v.abs().amax(-1, keepdim=True) / 448)
    return {"q_rot": q.view(-1, hq * d), "k": kp, "v": vp, "ks": ks, "vs": vs}
