"""The paged K/V cache's operators for sequences that share pages, as measured cases.

* ``attention``: causal grouped-query attention of a batch whose sequences share a long prefix of
  their cache (the same pages in their page tables), one layer's call. The block's rows (up to M per
  sequence) are rotated, written into the cache and attend to everything up to their own position.
* ``fork``: sequences made from one prompt (best-of-n sampling): each shares the prompt's pages, and the
  page that its next row falls into is copied, in every layer.
* ``copy``: a list of pages copied inside the pools, in every layer (what compaction moves).

``run`` computes them in elementary torch operations where ``own`` is false, and through
``layerstream_b200`` where it is true.
"""

import math
import random

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


# ---- cases ---------------------------------------------------------------------------------------


def _attention(name, heads, kv_heads, hd, dtype, page, groups, seqs, M, prefix, tail, ragged=False, rope=True, mix=1):
    return {"name": name, "op": "attention", "heads": heads, "kv_heads": kv_heads, "hd": hd, "dtype": dtype, "page": page,
            "groups": groups, "seqs": seqs, "M": M, "prefix": prefix, "tail": tail, "ragged": ragged, "rope": rope, "mix": mix}


def _fork(name, layers, kv_heads, hd, dtype, page, forks, n, M):
    return {"name": name, "op": "fork", "layers": layers, "kv_heads": kv_heads, "hd": hd, "dtype": dtype, "page": page,
            "forks": forks, "n": n, "M": M}


def _copy(name, layers, kv_heads, hd, dtype, page, pages, partial):
    return {"name": name, "op": "copy", "layers": layers, "kv_heads": kv_heads, "hd": hd, "dtype": dtype, "page": page,
            "pages": pages, "partial": partial}


def listed():
    return [
        # two samples of a short prompt, one token each: the call's latency (0.5B head layout)
        _attention("two short samples", 14, 2, 64, "f16", 64, 1, 2, 1, 128, 40),
        # best-of-16 of one 4k prompt, single tokens, answers of up to 300 tokens (0.5B head layout)
        _attention("16 samples of 4k", 14, 2, 64, "f16", 64, 1, 16, 1, 4096, 300),
        # a verify pass: 32 sequences under one 2k system prompt, 9 rows each (3B head layout)
        _attention("verify 32x9 over 2k", 16, 2, 128, "f16", 64, 1, 32, 9, 2048, 500),
        # four prompts of 8k sampled 16 times each, verify blocks of 5 (3B head layout, bf16 cache)
        _attention("4 prompts x 16, 8k", 16, 2, 128, "bf16", 256, 4, 64, 5, 8192, 700),
        # a 32k document asked 64 questions at once, single tokens, 8 kv heads
        _attention("64 readers of 32k", 32, 8, 128, "bf16", 64, 1, 64, 1, 32768, 900),
        # blocks of unequal length (some sequences idle) over small pages, rows rotated beforehand
        _attention("ragged, small pages", 6, 2, 64, "f16", 8, 2, 7, 5, 1000, 77, ragged=True, rope=False, mix=3),
        # prompts continued under a shared system prompt: 128-row prefill chunks of 8 sequences
        _attention("8 prefill chunks", 14, 2, 64, "f16", 64, 1, 8, 128, 4096, 260),
        # four samples of a short prompt: table work and a few tail rows (0.5B layout, 24 layers)
        _fork("fork 4", 24, 2, 64, "f16", 64, 4, 100, 1),
        # 63 samples of an 8k prompt with large pages (3B layout, 36 layers)
        _fork("fork 63, large pages", 36, 2, 128, "f16", 256, 63, 8136, 1),
        # the few pages that one rollback leaves to move
        _copy("copy 6 pages", 24, 2, 64, "f16", 64, 6, True),
        # compaction of a fragmented pool
        _copy("copy 1024 pages", 24, 2, 64, "f16", 64, 1024, False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "fork", "copy"])
    dtype = rng.choice(["f16", "bf16"])
    page = rng.choice([8, 16, 32, 64, 64, 128, 256])
    if op == "attention":
        heads, kv_heads, hd = rng.choice([(14, 2, 64), (16, 2, 128), (32, 8, 128), (6, 2, 64), (8, 8, 128), (12, 4, 64), (5, 1, 128)])
        while True:
            seqs = _log_int(rng, 2, 64)
            groups = rng.choice([1, 1, 1, min(2, seqs), min(5, seqs)])
            M = rng.choice([1, 1, 1, rng.randint(2, 33), rng.randint(2, 33), rng.randint(34, 128)])
            prefix = max(1, _log_int(rng, 64, 32768) // page) * page
            tail = _log_int(rng, 1, 1000)
            if seqs * (prefix + tail) * kv_heads * hd <= 64 * 33792 * 8 * 128 and seqs * M * heads * hd * (prefix + tail) <= 64 * 32 * 128 * 33792:
                break
        return {k: v for k, v in _attention("", heads, kv_heads, hd, dtype, page, groups, seqs, M, prefix, tail, rng.random() < 0.3,
                                            rng.random() < 0.7, rng.randint(0, 1 << 20)).items() if k != "name"}
    layers, kv_heads, hd = rng.choice([(24, 2, 64), (36, 2, 128), (2, 8, 128), (12, 4, 64)])
    row = layers * kv_heads * hd * 2 * 2
    if op == "fork":
        n = _log_int(rng, 1, 16384)
        forks = max(1, min(_log_int(rng, 1, 63), (1 << 29) // (row * page)))
        return {k: v for k, v in _fork("", layers, kv_heads, hd, dtype, page, forks, n, rng.choice([1, 1, rng.randint(2, 33)])).items() if k != "name"}
    pages = max(1, min(_log_int(rng, 1, 4096), (1 << 30) // (row * page)))
    return {k: v for k, v in _copy("", layers, kv_heads, hd, dtype, page, pages, rng.random() < 0.5).items() if k != "name"}


def _lengths(c):
    """Per sequence: cached positions before the block, and rows of the block."""
    pos0 = [c["prefix"] + (i * 7919 + c["mix"] * 31) % (c["tail"] + 1) for i in range(c["seqs"])]
    rows = [(i * 5 + c["mix"]) % (c["M"] + 1) if c["ragged"] else c["M"] for i in range(c["seqs"])]
    if c["ragged"]:
        rows[-1] = c["M"]
    return pos0, rows


def _group_of(c):
    return [i * c["groups"] // c["seqs"] for i in range(c["seqs"])]


def _fork_pages(c):
    """Whole pages that a fork shares, rows of the page it copies, and pages it holds of its own."""
    full, rest = divmod(c["n"], c["page"])
    return full, rest, -(-(c["n"] + c["M"]) // c["page"]) - full


def _copy_rows(c):
    return [(i * 37 + 11) % c["page"] + 1 if c["partial"] else c["page"] for i in range(c["pages"])]


def work(case):
    c = case
    if c["op"] == "attention":
        pos0, rows = _lengths(c)
        kv_row = c["kv_heads"] * c["hd"] * 2 * 2
        live = set(g for g, r in zip(_group_of(c), rows) if r)
        cached = len(live) * c["prefix"] + sum(p - c["prefix"] for p, r in zip(pos0, rows) if r)
        total = sum(rows)
        table = 8 * c["hd"] // 2 * total if c["rope"] else 0
        bytes_ = cached * kv_row + 2 * total * kv_row + 2 * total * c["heads"] * c["hd"] * 2 + table
        seen = sum(r * p + r * (r + 1) // 2 for p, r in zip(pos0, rows))
        return {"bytes": bytes_, "flops": 4 * c["hd"] * c["heads"] * seen}
    row = c["layers"] * c["kv_heads"] * c["hd"] * 2 * 2
    if c["op"] == "fork":
        full, rest, mine = _fork_pages(c)
        return {"bytes": row * rest * (c["forks"] + 1) + 4 * (full + 1 + c["forks"] * (full + mine)), "flops": 0}
    return {"bytes": 2 * row * sum(_copy_rows(c)) + 8 * c["pages"], "flops": 0}


# ---- inputs --------------------------------------------------------------------------------------


def _rope(hd, positions):
    """(cos, sin) pairs in 32 bits, angles in 64 bits."""
    inv = 1e6 ** (-torch.arange(0, hd, 2, dtype=torch.float64, device="cuda") / hd)
    ang = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()


def prepare(case, seed):
    c = case
    g = torch.Generator("cuda").manual_seed(seed)
    dt, page, kvh, hd = DTYPES[c["dtype"]], c["page"], c["kv_heads"], c["hd"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dt)

    def shuffled(n):
        return torch.randperm(n, generator=g, device="cuda")

    s = {"case": dict(c), "dt": dt}
    if c["op"] == "attention":
        pos0, rows = _lengths(c)
        group = _group_of(c)
        shared = c["prefix"] // page
        need = [-(-(p + r) // page) for p, r in zip(pos0, rows)]
        most = max(need)
        total = c["groups"] * shared + sum(n - shared for n in need)
        num_pages = total + 3  # a few pages that nobody names
        ids = shuffled(num_pages)[:total].tolist()
        prefixes = [ids[i * shared:(i + 1) * shared] for i in range(c["groups"])]
        at, tables = c["groups"] * shared, []
        for i, n in enumerate(need):
            tables.append(prefixes[group[i]] + ids[at:at + n - shared])
            at += n - shared
        s["layers"], s["layer"] = 2, 1
        s["k"], s["v"] = normal(2, kvh, num_pages, page, hd), normal(2, kvh, num_pages, page, hd)
        s["qkv"] = normal(c["seqs"] * c["M"], (c["heads"] + 2 * kvh) * hd)
        s["out"] = torch.zeros(c["seqs"] * c["M"], c["heads"] * hd, device="cuda", dtype=dt)
        s["rope"] = _rope(hd, max(pos0) + c["M"]) if c["rope"] else None
        s["tables"] = torch.tensor([t + [0] * (most - len(t)) for t in tables], dtype=torch.int32, device="cuda")
        s["pos0"] = torch.tensor(pos0, device="cuda")
        s["rows"] = torch.tensor(rows, device="cuda")
        s["context"] = max(p + r for p, r in zip(pos0, rows))
        if own:
            import layerstream_b200 as ls

            s["kv"] = ls.KvCache(s["k"].data_ptr(), s["v"].data_ptr(), layers=2, heads=c["heads"], kv_heads=kvh, hd=hd, page=page,
                                 num_pages=num_pages, seqs=c["seqs"], max_ctx=max(pos0) + c["M"], max_rows=c["seqs"] * c["M"], dtype=c["dtype"])
            for i, t in enumerate(tables):
                s["kv"].set_table(i, t, pos0[i])
            s["kv"].begin(rows, c["M"], torch.cuda.current_stream().cuda_stream)
        return s
    if c["op"] == "fork":
        full, rest, mine = _fork_pages(c)
        held, busy = full + (rest > 0), 1 + (c["n"] // page) // 4
        num_pages = held + busy + c["forks"] * mine + 5
        ids = shuffled(num_pages).tolist()
        most = -(-(c["n"] + c["M"]) // page)
        s["k"], s["v"] = normal(c["layers"], kvh, num_pages, page, hd), normal(c["layers"], kvh, num_pages, page, hd)
        # sequence 0 holds the prompt, the last one some other pages, those between are forked
        t = torch.full((c["forks"] + 2, max(most, busy)), -1, dtype=torch.int32, device="cuda")
        t[0, :held] = torch.tensor(ids[:held], dtype=torch.int32)
        t[-1, :busy] = torch.tensor(ids[held:held + busy], dtype=torch.int32)
        s["tables"] = t
        if own:
            import layerstream_b200 as ls

            kv = ls.KvCache(s["k"].data_ptr(), s["v"].data_ptr(), layers=c["layers"], heads=kvh, kv_heads=kvh, hd=hd, page=page,
                            num_pages=num_pages, seqs=c["forks"] + 2, max_ctx=max(most, busy) * page, max_rows=(c["forks"] + 2) * c["M"],
                            dtype=c["dtype"])
            kv.set_table(0, ids[:held], c["n"])
            kv.set_table(c["forks"] + 1, ids[held:held + busy], busy * page)
            s["kv"], s["counts"] = kv, [0] + [c["M"]] * c["forks"] + [0]
        return s
    num_pages = 2 * c["pages"] + 3
    ids = shuffled(num_pages)
    s["k"], s["v"] = normal(c["layers"], kvh, num_pages, page, hd), normal(c["layers"], kvh, num_pages, page, hd)
    s["src"], s["dst"] = ids[:c["pages"]].tolist(), ids[c["pages"]:2 * c["pages"]].tolist()
    s["rows"] = _copy_rows(c)
    return s


# ---- one pass ------------------------------------------------------------------------------------


def run(state):
    s, c = state, state["case"]
    if own:
        return _run_own(s, c)
    if c["op"] == "attention":
        return _plain_attention(s, c)
    if c["op"] == "fork":
        return _plain_fork(s, c)
    return _plain_copy(s, c)


def _run_own(s, c):
    import layerstream_b200 as ls

    stream = torch.cuda.current_stream().cuda_stream
    if c["op"] == "attention":
        s["kv"].attention(s["layer"], s["qkv"].data_ptr(), s["out"].data_ptr(), s["rope"].data_ptr() if c["rope"] else 0, stream=stream)
        return {"out": s["out"], "k": s["k"], "v": s["v"]}
    if c["op"] == "fork":
        s["kv"].fork(0, range(1, c["forks"] + 1), c["n"])
        s["kv"].begin(s["counts"], c["M"], stream)
        return {"tables": s["kv"].tables(), "k": s["k"], "v": s["v"]}
    ls.kv_copy_pages(s["k"].data_ptr(), s["v"].data_ptr(), c["layers"], c["kv_heads"], c["hd"], c["page"], s["k"].shape[2], s["src"], s["dst"],
                     s["rows"], stream=stream)
    return {"k": s["k"], "v": s["v"]}


def _rotated(x, table):
    """Rotate-half pairs (d, d + hd / 2) of x [seqs, M, heads, hd] by table [seqs, M, hd / 2, 2]."""
    cos, sin = table[..., 0].unsqueeze(2), table[..., 1].unsqueeze(2)
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_attention(s, c):
    n, M, H, kvh, hd, page = c["seqs"], c["M"], c["heads"], c["kv_heads"], c["hd"], c["page"]
    pos = s["pos0"][:, None] + torch.arange(M, device="cuda")  # [n, M]
    live = torch.arange(M, device="cuda") < s["rows"][:, None]
    x = s["qkv"].float().view(n, M, H + 2 * kvh, hd)
    q, k, v = x[:, :, :H], x[:, :, H:H + kvh], x[:, :, H + kvh:]
    if c["rope"]:
        table = s["rope"][pos]
        q, k = _rotated(q, table), _rotated(k, table)
    # the block's rows into their pages
    kp, vp = s["k"][s["layer"]].view(kvh, -1, hd), s["v"][s["layer"]].view(kvh, -1, hd)
    page_of = s["tables"].long().gather(1, (pos // page).clamp(max=s["tables"].shape[1] - 1))
    at = (page_of * page + pos % page)[live]
    kp[:, at] = k[live].transpose(0, 1).to(s["dt"])
    vp[:, at] = v[live].transpose(0, 1).to(s["dt"])
    # every sequence's context out of its pages
    p = torch.arange(s["context"], device="cuda")
    rows = s["tables"].long()[:, p // page] * page + p % page  # [n, context]
    held = p < (s["pos0"] + s["rows"])[:, None]
    K = kp[:, rows].float()  # [kvh, n, context, hd]
    V = vp[:, rows].float()
    V.mul_(held[None, :, :, None])
    qg = q.reshape(n, M, kvh, H // kvh, hd).permute(2, 0, 1, 3, 4).reshape(kvh, n, -1, hd)
    sc = (qg @ K.transpose(-1, -2) / math.sqrt(hd)).view(kvh, n, M, H // kvh, -1)
    sc.masked_fill_((p > pos[:, :, None])[None, :, :, None, :], -math.inf)
    w = (sc - sc.amax(-1, keepdim=True)).exp_()
    o = (w / w.sum(-1, keepdim=True)).view(kvh, n, M * (H // kvh), -1) @ V
    o = o.view(kvh, n, M, H // kvh, hd).permute(1, 2, 0, 3, 4).reshape(n, M, H * hd)
    s["out"].view(n, M, -1)[live] = o[live].to(s["dt"])
    return {"out": s["out"], "k": s["k"], "v": s["v"]}


def _plain_fork(s, c):
    full, rest, mine = _fork_pages(c)
    t, F = s["tables"], c["forks"]
    used = torch.zeros(s["k"].shape[2], dtype=torch.bool, device="cuda")
    kept = torch.cat([t[0], t[-1]])
    used[kept[kept >= 0].long()] = True
    free = (~used).nonzero()[:F * mine, 0].view(F, mine)  # the lowest free pages, fork by fork
    t[1:-1] = -1
    t[1:-1, :full] = t[0, :full]
    t[1:-1, full:full + mine] = free.int()
    if rest:
        for_all = t[0, full].long()
        s["k"][:, :, free[:, 0], :rest] = s["k"][:, :, for_all, :rest].unsqueeze(2)
        s["v"][:, :, free[:, 0], :rest] = s["v"][:, :, for_all, :rest].unsqueeze(2)
    return {"tables": t, "k": s["k"], "v": s["v"]}


def _plain_copy(s, c):
    src, dst = (torch.tensor(s[k], device="cuda") for k in ("src", "dst"))
    if c["partial"]:
        rows = torch.tensor(s["rows"], device="cuda")
        at = torch.arange(c["page"], device="cuda")
        moved = (at < rows[:, None])[None, None, :, :, None]
        s["k"][:, :, dst] = torch.where(moved, s["k"][:, :, src], s["k"][:, :, dst])
        s["v"][:, :, dst] = torch.where(moved, s["v"][:, :, src], s["v"][:, :, dst])
    else:
        s["k"][:, :, dst] = s["k"][:, :, src]
        s["v"][:, :, dst] = s["v"][:, :, src]
    return {"k": s["k"], "v": s["v"]}


# ---- the definition in 64 bits -------------------------------------------------------------------


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] == "attention":
        return _exact_attention(s, c)
    if c["op"] == "copy":
        for k in ("k", "v"):
            for i, j, r in zip(s["src"], s["dst"], s["rows"]):
                s[k][:, :, j, :r] = s[k][:, :, i, :r]
        return {"k": s["k"], "v": s["v"]}
    t = s["tables"].cpu().numpy().copy()
    taken = set(t[0].tolist()) | set(t[-1].tolist())
    free = iter(i for i in range(s["k"].shape[2]) if i not in taken)
    full, rest, mine = _fork_pages(c)
    for f in range(1, c["forks"] + 1):
        t[f, :full] = t[0, :full]
        for j in range(mine):
            t[f, full + j] = next(free)
        if rest:
            for k in ("k", "v"):
                s[k][:, :, int(t[f, full]), :rest] = s[k][:, :, int(t[0, full]), :rest]
    return {"tables": t, "k": s["k"], "v": s["v"]}


def _exact_attention(s, c):
    M, H, kvh, hd, page, layer = c["M"], c["heads"], c["kv_heads"], c["hd"], c["page"], s["layer"]
    G, half = H // kvh, hd // 2
    pos0, rows = _lengths(c)
    k64, v64, out = s["k"].double(), s["v"].double(), s["out"].double()
    for i in range(c["seqs"]):
        n, r = pos0[i], rows[i]
        if r == 0:
            continue
        pages = s["tables"][i].long()
        x = s["qkv"][i * M:i * M + r].double().view(r, H + 2 * kvh, hd)
        if c["rope"]:
            ang = s["rope"][n:n + r].double()[:, None]  # [r, 1, hd / 2, 2]
            turn = torch.complex(ang[..., 0], ang[..., 1])
            z = torch.complex(x[:, :H + kvh, :half], x[:, :H + kvh, half:]) * turn
            x = torch.cat([torch.cat([z.real, z.imag], -1), x[:, H + kvh:]], 1)
        for t in range(r):
            a, b = int(pages[(n + t) // page]), (n + t) % page
            k64[layer, :, a, b] = x[t, H:H + kvh]
            v64[layer, :, a, b] = x[t, H + kvh:]
        at = torch.arange(n + r, device="cuda")
        for g in range(kvh):
            K = s["k"][layer, g][pages[at // page], at % page].double()
            V = s["v"][layer, g][pages[at // page], at % page].double()
            K[n:] = x[:, H + g].to(s["dt"]).double()  # as the cache holds them
            V[n:] = x[:, H + kvh + g].to(s["dt"]).double()
            for t0 in range(0, r, 16):
                t1 = min(t0 + 16, r)
                e = n + t1
                sc = torch.einsum("thd,pd->thp", x[t0:t1, g * G:(g + 1) * G], K[:e]) / math.sqrt(hd)
                late = at[None, :e] > n + torch.arange(t0, t1, device="cuda")[:, None]
                sc = sc.masked_fill(late[:, None], -math.inf)
                o = torch.softmax(sc, -1) @ V[:e]
                out[i * M + t0:i * M + t1, g * G * hd:(g + 1) * G * hd] = o.reshape(t1 - t0, G * hd)
    return {"out": out, "k": k64, "v": v64}


if __name__ == "__main__":
    for case in listed() + [draw(random.Random(0))]:
        print(case, work(case))
