"""Measured operators of the paged key / value cache and of the attention that reads it.

A cache holds pages ``[layers, pages, kv heads, page tokens, head dim]`` for K and for V, a page table ``[slots, pages
of a slot]`` (-1: none), the length of each slot and a count of the slots that hold each page.  Five operators:

attend   queries ``[n, Hq, T, D]`` (the last T tokens of n sequences) over the sequences' pages.  Sequences of a group
         share the pages of a prefix.  Key j is visible to query t where j < length - (T - 1 - t).
copy     whole pages of all layers, from a list of pages to another
refork   samples that ended give their pages back, and samples that go on are forked into their slots: full pages are
         shared, the page that is still being filled is copied
admit    ended sequences give their pages back, new ones claim pages and their keys and values are written
compact  the pages in use move to the front of the pool, tables and counts follow

Each case is one call (or the short run of calls named above) as a serving program makes it.  ``own = False`` computes
the plain form with elementary torch operations.
"""

import math

import torch

own = False

E4M3_MAX = 448.0


# --------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # a chat with one user: one sequence, one token, nothing shared; latency counts
        dict(name="attend 1 seq", op="attend", n=1, groups=1, t=1, hq=32, hkv=8, d=64, page=16, prefix=0, suffix=1000, q="float16", kv="float16"),
        # 32 samples of one 8k prompt, each some hundred tokens on
        dict(name="attend 32 of 8k", op="attend", n=32, groups=1, t=1, hq=32, hkv=8, d=128, page=16, prefix=8219, suffix=600, q="bfloat16", kv="bfloat16"),
        # six prompts with eight samples each over an 8-bit cache
        dict(name="attend 6x8 of 4k e4m3", op="attend", n=48, groups=6, t=1, hq=32, hkv=8, d=128, page=32, prefix=4131, suffix=700, q="bfloat16", kv="float8_e4m3fn"),
        # 128 samples of a 32k document, three drafted tokens verified with the next one
        dict(name="attend 128x4 of 32k", op="attend", n=128, groups=1, t=4, hq=32, hkv=8, d=128, page=64, prefix=32768, suffix=1024, q="bfloat16", kv="bfloat16"),
        # one page changes its place
        dict(name="copy 1 page", op="copy", n=1, layers=2, pages=64, hkv=8, d=128, page=16, kv="bfloat16"),
        # a part of the pool is moved aside, all 32 layers of it
        dict(name="copy 250 pages", op="copy", n=250, layers=32, pages=640, hkv=8, d=128, page=16, kv="bfloat16"),
        # four samples of one short prompt
        dict(name="refork 4", op="refork", n=4, parents=1, length=300, layers=2, pages=256, slots=16, hkv=8, d=128, page=16, kv="bfloat16"),
        # 256 samples of 16 prompts of about 4k tokens, four layers in this pool
        dict(name="refork 256 of 16", op="refork", n=256, parents=16, length=4093, layers=4, pages=12000, slots=300, hkv=8, d=128, page=16, kv="bfloat16"),
        # eight sequences that begin with one token each
        dict(name="admit 8x1", op="admit", n=8, length=1, pages=256, slots=16, hkv=8, d=128, page=16, kv="bfloat16"),
        # 32 prompts of up to 2k tokens enter an 8-bit cache
        dict(name="admit 32x2k e4m3", op="admit", n=32, length=2011, pages=9000, slots=64, hkv=8, d=128, page=16, kv="float8_e4m3fn"),
        # a small pool with holes
        dict(name="compact 200", op="compact", layers=1, pages=200, slots=16, hkv=8, d=64, page=16, kv="float16"),
        # a large pool, a third in use
        dict(name="compact 16k", op="compact", layers=4, pages=16001, slots=256, hkv=8, d=128, page=16, kv="bfloat16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "copy", "refork", "admit", "compact"])
    page = rng.choice([16, 32, 64, 128])
    d = rng.choice([64, 128])
    kv = rng.choice(["bfloat16", "float16", "float8_e4m3fn"])
    if op == "attend":
        hq, hkv = rng.choice([(32, 8), (32, 8), (16, 16), (8, 1), (28, 4), (64, 4), (12, 3)])
        q = rng.choice(["bfloat16", "float16"]) if kv == "float8_e4m3fn" else kv
        n = _log(rng, 1, 128)
        c = dict(op=op, n=n, groups=rng.randint(1, min(n, 8)), t=rng.choice([1, 1, 1, 2, 3, 5, 8]), hq=hq, hkv=hkv, d=d, page=page,
                 prefix=rng.choice([0, 1, 1, 1]) * _log(rng, 20, 32768), suffix=_log(rng, 8, 8192), q=q, kv=kv)
        while n * hkv * d * (c["prefix"] + c["suffix"]) > 128 * 8 * 128 * 33792 or n * c["t"] * hq * d * (c["prefix"] + c["suffix"]) > 512 * 32 * 128 * 33792:
            c["prefix"], c["suffix"] = c["prefix"] // 2, max(8, c["suffix"] // 2)
        return c
    hkv = rng.choice([1, 2, 3, 8])
    layers = _log(rng, 1, 32)
    if op == "copy":
        n = _log(rng, 1, 256)
        per = 2 * layers * hkv * d * page * (1 if kv == "float8_e4m3fn" else 2)
        n = max(1, min(n, 500 * 2 ** 20 // per))
        return dict(op=op, n=n, layers=layers, pages=2 * n + rng.randint(1, 2 * n + 8), hkv=hkv, d=d, page=page, kv=kv)
    if op == "refork":
        n, length = _log(rng, 1, 256), _log(rng, 1, 4096)
        parents = rng.randint(1, min(n, 16))
        pages = parents * -(-length // page) + 3 * n + rng.randint(1, 500)
        layers = max(1, min(layers, 2 ** 32 // (pages * hkv * d * page * 4)))
        return dict(op=op, n=n, parents=parents, length=length, layers=layers, pages=pages, slots=n + parents + rng.randint(0, 40), hkv=hkv, d=d, page=page, kv=kv)
    if op == "admit":
        n, length = _log(rng, 1, 256), _log(rng, 1, 2048)
        length = max(1, min(length, 32 * 2011 // n))
        return dict(op=op, n=n, length=length, pages=2 * n * -(-length // page) + rng.randint(1, 600), slots=n + rng.randint(0, 40), hkv=hkv, d=d, page=page, kv=kv)
    pages = _log(rng, 20, 16000)
    while layers > 1 and layers * pages * hkv * d * page > 4 * 16000 * 8 * 128 * 16:
        layers //= 2
    while layers * pages * hkv * d * page > 4 * 16000 * 8 * 128 * 16:
        pages //= 2
    return dict(op=op, layers=layers, pages=pages, slots=rng.randint(4, 256), hkv=hkv, d=d, page=page, kv=kv)


# --------------------------------------------------------------------------------------------------- sizes
def _dtype(name):
    return getattr(torch, name)


def _size(name):
    return 1 if name == "float8_e4m3fn" else 2


def _spread(n, top):
    """n whole numbers in 1..top that do not rise or fall with their index; the first is top."""
    return [top - (i * 7919) % top for i in range(n)]


def _members(c):
    """Sequences of each group: nearly equal numbers."""
    n, g = c["n"], c["groups"]
    return [n // g + (i < n % g) for i in range(g)]


def _lens(c):
    """Length of each sequence and shared length of each group; a group's prefix is a little shorter than the one before it.
    Every sequence holds its T newest tokens behind the shared pages."""
    suffix = [max(c["t"], s) for s in _spread(c["n"], c["suffix"])]
    prefix = [max(0, c["prefix"] - 37 * i) for i in range(c["groups"])]
    shared = [p // c["page"] * c["page"] for p in prefix]
    lens, i = [], 0
    for g, m in enumerate(_members(c)):
        lens += [prefix[g] + suffix[i + j] for j in range(m)]
        i += m
    return lens, shared


def _live(c):
    """Which pages of a pool with holes are in use: a third, spread by a rule."""
    return [(p * 40503 + (p >> 3) * 977) % 1000 < 333 for p in range(c["pages"])]


def work(c):
    if c["op"] == "attend":
        lens, shared = _lens(c)
        tokens, i = 0, 0
        for g, m in enumerate(_members(c)):
            tokens += shared[g] + sum(lens[i + j] - shared[g] for j in range(m))
            i += m
        rows = c["n"] * c["t"] * c["hq"]
        pairs = sum(sum(max(0, n - (c["t"] - 1 - t)) for t in range(c["t"])) for n in lens) * c["hq"]
        return {"bytes": 2 * tokens * c["hkv"] * c["d"] * _size(c["kv"]) + rows * (2 * c["d"] * 2 + 4), "flops": 4 * c["d"] * pairs}
    token = 2 * c.get("layers", 1) * c["hkv"] * c["d"] * _size(c["kv"])  # K and V of one token, all layers
    if c["op"] == "copy":
        return {"bytes": 2 * c["n"] * c["page"] * token + 8 * c["n"], "flops": 0}
    if c["op"] == "refork":
        lens = _spread(c["parents"], c["length"])
        by = [lens[i % c["parents"]] for i in range(c["n"])]
        tables = sum(4 * 4 * -(-x // c["page"]) for x in by)  # entries read and written, counts read and written
        return {"bytes": sum(2 * (x % c["page"]) * token for x in by) + tables, "flops": 0}
    if c["op"] == "admit":
        lens = _spread(c["n"], c["length"])
        return {"bytes": sum(lens) * (token + 2 * c["hkv"] * c["d"] * 2) + sum(3 * 4 * -(-x // c["page"]) for x in lens), "flops": 0}
    live = _live(c)
    moved = sum(live[sum(live):])
    return {"bytes": 2 * moved * c["page"] * token + 2 * 4 * c["pages"] + 2 * 4 * sum(live), "flops": 0}


# --------------------------------------------------------------------------------------------------- inputs
def _random(gen, shape, dtype, scale=None):
    """Normal values of a type; codes of the 8-bit type stand for normal values divided by their head's scale."""
    out = torch.empty(shape, dtype=dtype, device="cuda")
    for part in out.flatten(0, 1).split(max(1, 2 ** 27 // max(1, out[0, 0].numel()))) if out.ndim == 5 else [out]:
        x = torch.randn(part.shape, generator=gen, device="cuda")
        if scale is not None:
            x = (x / scale[0].view(-1, 1, 1)).clamp(-E4M3_MAX, E4M3_MAX)
        part.copy_(x.to(dtype))
    return out


def _pool(c, gen, layers, pages):
    kv = _dtype(c["kv"])
    s = {"k_scale": None, "v_scale": None}
    if c["kv"] == "float8_e4m3fn":  # one dequantisation factor for each layer and kv head
        for x in ("k_scale", "v_scale"):
            s[x] = (0.008 + 0.004 * torch.rand(1, c["hkv"], generator=gen, device="cuda")).expand(layers, -1).contiguous()
    shape = (layers, pages, c["hkv"], c["page"], c["d"])
    s["k"] = _random(gen, shape, kv, s["k_scale"])
    s["v"] = _random(gen, shape, kv, s["v_scale"])
    return s


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def prepare(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    page = c["page"]
    if c["op"] == "attend":
        lens, shared = _lens(c)
        width = max(-(-n // page) for n in lens) + 1
        rows, ref, i, at = [], [], 0, 0
        for g, m in enumerate(_members(c)):
            common = list(range(at, at + shared[g] // page))
            at += len(common)
            ref += [m] * len(common)
            for j in range(m):
                mine = -(-lens[i + j] // page) - len(common)
                rows.append(common + list(range(at, at + mine)) + [-1] * (width - len(common) - mine))
                ref += [1] * mine
                at += mine
            i += m
        pages = at + 5
        order = torch.randperm(pages, generator=host).to(torch.int32)  # pages were claimed and given back in any order
        table = torch.tensor(rows, dtype=torch.int64)
        table = torch.where(table >= 0, order[table.clamp(min=0)], -1)
        counts = torch.zeros(pages, dtype=torch.int32)
        counts[order[:at].long()] = torch.tensor(ref, dtype=torch.int32)
        s = _pool(c, gen, 1, pages)
        ends = [0]
        for m in _members(c):
            ends.append(ends[-1] + m)
        return s | {"op": "attend", "page_table": table.to(torch.int32).cuda(), "seq_lens": _ints(lens), "ref_counts": counts.cuda(),
                    "q": _random(gen, (c["n"], c["hq"], c["t"], c["d"]), _dtype(c["q"])), "groups": _ints(ends) if c["prefix"] else None, "shared": _ints(shared) if c["prefix"] else None}
    if c["op"] == "copy":
        s = _pool(c, gen, c["layers"], c["pages"])
        order = torch.randperm(c["pages"], generator=host).to(torch.int32).cuda()
        return s | {"op": "copy", "src": order[:c["n"]].clone(), "dst": order[c["n"]:2 * c["n"]].clone(),
                    "page_table": _ints([[-1]]), "seq_lens": _ints([0]), "ref_counts": torch.zeros(c["pages"], dtype=torch.int32, device="cuda")}
    if c["op"] == "refork":
        # slots: the parents, then the samples of the step before, which hang on other parents
        p, n = c["parents"], c["n"]
        lens = _spread(p, c["length"])
        width = -(-c["length"] // page) + 1
        table, ref = torch.full((c["slots"], width), -1, dtype=torch.int32), torch.zeros(c["pages"], dtype=torch.int32)
        order = torch.randperm(c["pages"], generator=host).to(torch.int32)
        seq, at = torch.zeros(c["slots"], dtype=torch.int32), 0
        slots = torch.randperm(c["slots"], generator=host).to(torch.int32)
        for i in range(p):
            k = -(-lens[i] // page)
            table[slots[i], :k] = order[at:at + k]
            ref[order[at:at + k].long()] = 1
            seq[slots[i]] = lens[i]
            at += k
        for i in range(n):
            parent, child, x = slots[(i + 1) % p], slots[p + i], lens[(i + 1) % p]
            full, part = x // page, x % page
            table[child, :full] = table[parent, :full]
            ref[table[parent, :full].long()] += 1
            if part:
                table[child, full] = order[at]
                ref[order[at]] = 1
                at += 1
            seq[child] = x
        parents = slots[:p][torch.arange(n) % p]
        return _pool(c, gen, c["layers"], c["pages"]) | {
            "op": "refork", "page_table": table.cuda(), "seq_lens": seq.cuda(), "ref_counts": ref.cuda(), "parents": parents.cuda(), "children": slots[p:p + n].clone().cuda()}
    if c["op"] == "admit":
        n, lens = c["n"], _spread(c["n"], c["length"])
        width = -(-c["length"] // page) + 1
        table, ref = torch.full((c["slots"], width), -1, dtype=torch.int32), torch.zeros(c["pages"], dtype=torch.int32)
        order = torch.randperm(c["pages"], generator=host).to(torch.int32)
        seq, at = torch.zeros(c["slots"], dtype=torch.int32), 0
        slots = torch.randperm(c["slots"], generator=host).to(torch.int32)
        for i in range(c["slots"]):  # all slots are taken: the n that ended, and the others
            x = lens[(i + 1) % n] if i < n else 1
            k = -(-x // page)
            if at + k > c["pages"] - sum(-(-y // page) for y in lens) // 2:
                break
            table[slots[i], :k] = order[at:at + k]
            ref[order[at:at + k].long()] = 1
            seq[slots[i]] = x
            at += k
        s = _pool(c, gen, 1, c["pages"])
        dtype = torch.float16 if c["kv"] == "float16" else torch.bfloat16
        shape = (n, c["hkv"], c["length"], c["d"])
        return s | {"op": "admit", "page_table": table.cuda(), "seq_lens": seq.cuda(), "ref_counts": ref.cuda(), "seqs": slots[:n].clone().cuda(), "n_new": _ints(lens),
                    "k_new": _random(gen, shape, dtype), "v_new": _random(gen, shape, dtype)}
    live = torch.tensor(_live(c)).nonzero().flatten().to(torch.int32)
    live = live[torch.randperm(len(live), generator=host)]
    per = -(-len(live) // c["slots"])
    table, seq = torch.full((c["slots"], per + 1), -1, dtype=torch.int32), torch.zeros(c["slots"], dtype=torch.int32)
    ref = torch.zeros(c["pages"], dtype=torch.int32)
    for i in range(c["slots"]):
        mine = live[i * per:(i + 1) * per]
        table[i, :len(mine)] = mine
        seq[i] = max(0, len(mine) * page - i % page)
        ref[mine.long()] = 1
    return _pool(c, gen, c["layers"], c["pages"]) | {"op": "compact", "page_table": table.cuda(), "seq_lens": seq.cuda(), "ref_counts": ref.cuda(),
                                                     "page_table_before": table.cuda(), "ref_counts_before": ref.cuda()}


# --------------------------------------------------------------------------------------------------- one pass
def run(s):
    return _calls(s) if own else _plain(s)


def _calls(s):
    """The calls a user makes.  The cache object is the handle a program opens once over its tensors."""
    c = s.get("cache")
    if c is None:
        import sys

        if "fp4-fa4_b200" not in sys.path:
            sys.path.insert(0, "fp4-fa4_b200")
        from fa4b import PagedKVCache

        c = s["cache"] = PagedKVCache(s["k"], s["v"], s["page_table"], s["seq_lens"], s["ref_counts"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    if s["op"] == "attend":
        out, lse = c.attend(s["q"], group_offsets=s["groups"], shared_lens=s["shared"])
        return {"out": out, "lse": lse}
    if s["op"] == "copy":
        c.copy_pages(s["src"], s["dst"])
        return {"k": c.k, "v": c.v}
    if s["op"] == "refork":
        c.free(s["children"])
        c.fork(s["parents"], s["children"])
    elif s["op"] == "admit":
        c.free(s["seqs"])
        c.extend(s["seqs"], s["n_new"])
        c.write(s["k_new"], s["v_new"], s["seqs"], n_new=s["n_new"])
    else:  # the tables and counts of the pool with holes come back first, so that each pass does the same work
        c.page_table.copy_(s["page_table_before"])
        c.ref_counts.copy_(s["ref_counts_before"])
        c.compact()
    return {"k": c.k, "v": c.v, "page_table": c.page_table, "seq_lens": c.seq_lens, "ref_counts": c.ref_counts}


def _plain(s):
    if s["op"] == "attend":
        return _plain_attend(s)
    k, v, table, lens, ref = s["k"], s["v"], s["page_table"], s["seq_lens"], s["ref_counts"]
    kb, vb = (k.view(torch.uint8), v.view(torch.uint8)) if k.dtype == torch.float8_e4m3fn else (k, v)
    page = k.shape[3]
    if s["op"] == "copy":
        src, dst = s["src"].long(), s["dst"].long()
        kb[:, dst] = kb[:, src]
        vb[:, dst] = vb[:, src]
        return {"k": k, "v": v}
    column = torch.arange(table.shape[1], device=table.device)
    if s["op"] == "refork":
        _plain_free(s["children"].long(), table, lens, ref)
        parents, children = s["parents"].long(), s["children"].long()
        x = lens[parents].long()
        full, part = x // page, x % page
        need = (part > 0).long()
        spare = (ref == 0).nonzero().flatten()
        fresh = spare[(need.cumsum(0) - need).clamp(max=len(spare) - 1)]
        rows = table[parents]
        tail = rows.gather(1, full.clamp(max=table.shape[1] - 1)[:, None]).flatten().long()
        held = column < full[:, None]
        ref.index_add_(0, rows[held].long(), torch.ones_like(rows[held]))
        take = need > 0
        ref[fresh[take]] = 1
        rows = torch.where(column == full[:, None], torch.where(take, fresh, -1)[:, None].to(torch.int32), torch.where(held, rows, -1))
        table[children] = rows
        lens[children] = x.to(torch.int32)
        src, dst, ok = tail[take], fresh[take], (torch.arange(page, device=k.device) < part[take][:, None])[None, :, None, :, None]
        kb[:, dst] = torch.where(ok, kb[:, src], kb[:, dst])
        vb[:, dst] = torch.where(ok, vb[:, src], vb[:, dst])
    elif s["op"] == "admit":
        seqs, new = s["seqs"].long(), s["n_new"].long()
        _plain_free(seqs, table, lens, ref)
        held = (lens[seqs].long() + page - 1) // page
        need = (lens[seqs].long() + new + page - 1) // page - held
        spare = (ref == 0).nonzero().flatten()
        at = column - held[:, None]
        mine = (at >= 0) & (at < need[:, None])
        fresh = spare[((need.cumsum(0) - need)[:, None] + at).clamp(0, len(spare) - 1)]
        table[seqs] = torch.where(mine, fresh.to(torch.int32), table[seqs])
        ref[fresh[mine]] = 1
        lens[seqs] += new.to(torch.int32)
        kn, vn = s["k_new"], s["v_new"]
        t = torch.arange(kn.shape[2], device=k.device)
        which, tok = (t < new[:, None]).nonzero(as_tuple=True)
        pos = lens[seqs][which].long() - new[which] + tok
        pg, slot = table[seqs[which], pos // page].long(), pos % page
        k[0].view(kb.dtype)[pg, :, slot] = _plain_store(kn[which, :, tok], s["k_scale"], k.dtype).view(kb.dtype)
        v[0].view(vb.dtype)[pg, :, slot] = _plain_store(vn[which, :, tok], s["v_scale"], v.dtype).view(vb.dtype)
    else:
        table.copy_(s["page_table_before"])
        ref.copy_(s["ref_counts_before"])
        live = ref > 0
        n = live.sum()
        index = torch.arange(len(ref), device=ref.device)
        src = (live & (index >= n)).nonzero().flatten()
        dst = (~live & (index < n)).nonzero().flatten()
        kb[:, dst] = kb[:, src]
        vb[:, dst] = vb[:, src]
        to = index.to(torch.int32)
        to[src] = dst.to(torch.int32)
        table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()], table))
        ref[dst] = ref[src]
        ref[src] = 0
    return {"k": k, "v": v, "page_table": table, "seq_lens": lens, "ref_counts": ref}


def _plain_free(seqs, table, lens, ref):
    rows = table[seqs]
    pages = rows[rows >= 0].long()
    ref.index_add_(0, pages, torch.full_like(pages, -1, dtype=torch.int32))
    table[seqs] = -1
    lens[seqs] = 0


def _plain_store(x, scale, dtype):
    if scale is None:
        return x.to(dtype)
    return (x.float() / scale[0][None, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(dtype)


def _plain_attend(s):
    q, table, lens = s["q"], s["page_table"], s["seq_lens"]
    n, hq, t, d = q.shape
    _, _, hkv, page, _ = s["k"].shape
    at = table.clamp(min=0).long()

    def dense(pool, scale):
        x = pool[0][at].float()  # [n, pages, hkv, page, d]
        if scale is not None:
            x = x * scale[0][None, None, :, None, None]
        return x.transpose(1, 2).reshape(n, hkv, -1, d)

    keys = torch.arange(table.shape[1] * page, device=q.device)
    last = lens[:, None] - (t - 1 - torch.arange(t, device=q.device))  # [n, t]
    seen = (keys < last[:, :, None])[:, None, None]
    x = q.float().view(n, hkv, hq // hkv, t, d).reshape(n, hkv, -1, d)
    scores = (x @ dense(s["k"], s["k_scale"]).transpose(-1, -2)).view(n, hkv, hq // hkv, t, -1) * d ** -0.5
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    values = dense(s["v"], s["v_scale"]).masked_fill((keys >= lens[:, None])[:, None, :, None], 0)
    out = (p.view(n, hkv, -1, len(keys)) @ values).view(n, hkv, hq // hkv, t, d) / total.clamp(min=1e-30)
    lse = top + torch.log(total)
    lse = lse.masked_fill(total == 0, -math.inf)
    return {"out": out.view(n, hq, t, d).to(q.dtype), "lse": lse.view(n, hq, t)}


# --------------------------------------------------------------------------------------------------- in 64 bits
def exact(c, seed):
    s = prepare(c, seed)
    page = c["page"]
    if c["op"] == "attend":
        n, hq, t, d = s["q"].shape
        hkv = c["hkv"]
        out = torch.zeros(n, hq, t, d, dtype=torch.float64, device="cuda")
        lse = torch.full((n, hq, t), -math.inf, dtype=torch.float64, device="cuda")
        for i in range(n):
            total = int(s["seq_lens"][i])
            pages = s["page_table"][i, :-(-total // page)].long()
            keys = s["k"][0, pages].double().permute(1, 0, 2, 3).flatten(1, 2)[:, :total]
            values = s["v"][0, pages].double().permute(1, 0, 2, 3).flatten(1, 2)[:, :total]
            if s["k_scale"] is not None:
                keys, values = keys * s["k_scale"][0].double()[:, None, None], values * s["v_scale"][0].double()[:, None, None]
            for j in range(t):
                m = total - (t - 1 - j)
                if m <= 0:
                    continue
                z = torch.einsum("hgd,hkd->hgk", s["q"][i, :, j].double().view(hkv, hq // hkv, d), keys[:, :m]) / math.sqrt(d)
                out[i, :, j] = torch.einsum("hgk,hkd->hgd", torch.softmax(z, -1), values[:, :m]).reshape(hq, d)
                lse[i, :, j] = torch.logsumexp(z, -1).reshape(hq)
        return {"out": out, "lse": lse}
    # page by page and token by token, on lists
    table, lens, ref = s["page_table"].tolist(), s["seq_lens"].tolist(), s["ref_counts"].tolist()
    pools = [s[x].double() for x in ("k", "v")]

    def move(src, dst, tokens):
        for p in pools:
            p[:, dst, :, :tokens] = p[:, src, :, :tokens].clone()

    def drop(slot):
        for x in table[slot]:
            if x >= 0:
                ref[x] -= 1
        table[slot], lens[slot] = [-1] * len(table[slot]), 0

    def claim():
        x = ref.index(0)
        ref[x] = 1
        return x

    if c["op"] == "copy":
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            move(a, b, page)
        return {"k": pools[0], "v": pools[1]}
    if c["op"] == "refork":
        for x in s["children"].tolist():
            drop(x)
        for a, b in zip(s["parents"].tolist(), s["children"].tolist()):
            full, part = divmod(lens[a], page)
            for j in range(full):
                table[b][j] = table[a][j]
                ref[table[a][j]] += 1
            if part:
                table[b][full] = claim()
                move(table[a][full], table[b][full], part)
            lens[b] = lens[a]
    elif c["op"] == "admit":
        for x in s["seqs"].tolist():
            drop(x)
        for i, (x, new) in enumerate(zip(s["seqs"].tolist(), s["n_new"].tolist())):
            for j in range(-(-lens[x] // page), -(-(lens[x] + new) // page)):
                table[x][j] = claim()
            first, lens[x] = lens[x], lens[x] + new
            for j in range(first // page, -(-lens[x] // page)):
                a, b = max(first, j * page), min(lens[x], (j + 1) * page)
                for p, y, z in ((pools[0], s["k_new"], s["k_scale"]), (pools[1], s["v_new"], s["v_scale"])):
                    y = y[i, :, a - first:b - first].double()
                    p[0, table[x][j], :, a - j * page:b - j * page] = y if z is None else (y / z[0].double()[:, None, None]).clamp(-E4M3_MAX, E4M3_MAX)
    else:
        n = sum(x > 0 for x in ref)
        holes = [p for p in range(n) if ref[p] == 0]
        to = {}
        for p in range(n, len(ref)):
            if ref[p] > 0:
                to[p] = holes[len(to)]
                move(p, to[p], page)
                ref[to[p]], ref[p] = ref[p], 0
        table = [[to.get(x, x) for x in row] for row in table]
    return {"k": pools[0], "v": pools[1], "page_table": _ints(table), "seq_lens": _ints(lens), "ref_counts": _ints(ref)}
