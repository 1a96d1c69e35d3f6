"""Attention over a paged cache against the definition in 64 bits.

Tolerances, with u = half a step of the 16-bit type (2^-8 bf16, 2^-11 f16), A = sum_j softmax_j |v_j|:
  scores   products of 16-bit values are exact, sums of D = 64 or 128 of them are taken in groups of 16 with at most
           2^-22 of the group's magnitudes lost each: e = 2^-19 max_j scale sum_d |q_d k_jd|
  lse      e, 2^-22 per exponential and at most 64 additions in a row of 2^-24 each: 2^-18, and 2^-22 |lse| for the
           logarithm and its scaling
  out      every probability is off by u (rounded for the product) + 2 e + 2^-17 (exponential and sum): A (u + 2 e + 2^-17);
           the result is rounded: u |out|; below the type's normal range steps are absolute: a probability in f16 is off
           by at most 2^-25 of a row maximum that counts at least 1, n keys of them: n 2^-25 max |v|
An E4M3 cache computes in f16 whatever the queries are, its probabilities have u = 2^-11; the product with v_scale is one
more 32-bit rounding, inside 2^-17."""

import math
import random

import pytest
import torch

from fa4b import PagedKVCache

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, E4 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
U = {BF: 2.0 ** -8, HF: 2.0 ** -11}


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def build(lens, shared, members, *, page=16, hkv=2, d=128, dtype=BF, layers=1, seed=0, spare_pages=3, shuffle_slots=True, width=None, amp=1.0):
    """A cache of sequences in groups.  Tokens that are not there are NaN.  Returns (cache, slots, offsets)."""
    rng = random.Random(seed)
    gen = torch.Generator().manual_seed(seed)
    n = len(lens)
    width = width or max([-(-x // page) for x in lens] + [1]) + 1
    slots = list(range(n + 2))
    if shuffle_slots:
        rng.shuffle(slots)
    rows, pages_used, i = [], 0, 0
    for m, sh in zip(members, shared):
        full = sh // page
        common = list(range(pages_used, pages_used + full))
        pages_used += full
        for j in range(m):
            mine = max(0, -(-lens[i] // page) - full)
            rows.append(common[:-(-lens[i] // page)] + list(range(pages_used, pages_used + mine)))
            pages_used += mine
            i += 1
    for _ in range(n - i):  # rows behind the last group
        mine = -(-lens[i] // page)
        rows.append(list(range(pages_used, pages_used + mine)))
        pages_used += mine
        i += 1
    total = max(1, pages_used) + spare_pages
    order = torch.randperm(total, generator=gen)
    table = torch.full((n + 2, width), -1, dtype=torch.int32)
    seq = torch.zeros(n + 2, dtype=torch.int32)
    refs = torch.zeros(total, dtype=torch.int32)
    k, v = [(amp * torch.randn(layers, total, hkv, page, d, generator=gen)).to(dtype) for _ in range(2)]
    written = torch.zeros(total, page, dtype=torch.bool)
    for i, row in enumerate(rows):
        p = order[torch.tensor(row, dtype=torch.long)]
        table[slots[i], :len(row)] = p.to(torch.int32)
        seq[slots[i]] = lens[i]
        refs[p] += 1
        for j, x in enumerate(p.tolist()):
            written[x, :max(0, min(page, lens[i] - j * page))] = True
    hole = ~written[None, :, None, :, None]
    scales = {}
    if dtype == E4:
        scales = {x: (0.05 + 0.2 * torch.rand(layers, hkv, generator=gen)).to(DEV) for x in ("k_scale", "v_scale")}
        for t in (k, v):
            t.view(torch.uint8).masked_fill_(hole, 0x7f)
    else:
        for t in (k, v):
            t.masked_fill_(hole, float("nan"))
    c = PagedKVCache(k.to(DEV), v.to(DEV), table.to(DEV), seq.to(DEV), refs.to(DEV), **scales)
    offsets = [0]
    for m in members:
        offsets.append(offsets[-1] + m)
    return c, slots[:n], offsets


def queries(n, hq, t, d, dtype, seed, amp=1.0):
    gen = torch.Generator().manual_seed(1000 + seed)
    return (amp * torch.randn(n, hq, t, d, generator=gen)).to(dtype).to(DEV)


def compare(c, q, out, lse, slots, *, layer=0, scale=None, rows=None, holes=()):
    """Every row against the definition; `holes`: (row, key) pairs that do not exist."""
    n, hq, t, d = q.shape
    hkv, page = c.k.shape[2], c.k.shape[3]
    scale = scale or d ** -0.5
    u = U[q.dtype]
    up = 2.0 ** -11 if c.k.dtype == E4 else u
    table, lens = c.page_table.cpu(), c.seq_lens.cpu().tolist()
    for i in range(n) if rows is None else rows:
        length = lens[slots[i]] if 0 <= slots[i] < len(lens) else 0
        m = -(-length // page)
        pages = table[slots[i], :m].long().to(DEV) if m else torch.empty(0, dtype=torch.long, device=DEV)
        k, v = (x[layer, pages.clamp(min=0, max=x.shape[1] - 1)].double().permute(1, 0, 2, 3).reshape(hkv, -1, d)[:, :length] for x in (c.k, c.v))
        if c.k_scale is not None:
            k, v = k * c.k_scale[layer].double()[:, None, None], v * c.v_scale[layer].double()[:, None, None]
        gone = torch.zeros(length, dtype=torch.bool, device=DEV)
        for r, key in holes:
            if r == i:
                gone[key] = True
        for j in range(t):
            keys = torch.arange(length, device=DEV)[: max(0, length - (t - 1 - j))]
            keys = keys[~gone[keys]]
            o, s = out[i, :, j].double(), lse[i, :, j].double()
            if len(keys) == 0:
                assert (o == 0).all() and (s == -math.inf).all(), (i, j)
                continue
            kk, vv = k[:, keys], v[:, keys]
            x = q[i, :, j].double().view(hkv, -1, d)
            z = scale * x @ kk.transpose(1, 2)
            e = 2.0 ** -19 * scale * (x.abs() @ kk.abs().transpose(1, 2)).amax(-1)
            w = torch.softmax(z, -1)
            want, want_lse = (w @ vv), torch.logsumexp(z, -1)
            a = w @ vv.abs()
            tol = a * (up + 2 * e[..., None] + 2.0 ** -17) + want.abs() * u + len(keys) * 2.0 ** -25 * vv.abs().amax() + 2.0 ** -25
            off = (o.view(hkv, -1, d) - want).abs()
            assert (off <= tol).all(), (i, j, (off / tol).max().item(), (off / tol).argmax().item())
            off = (s.view(hkv, -1) - want_lse).abs()
            tol = e + 2.0 ** -18 + 2.0 ** -22 * want_lse.abs()
            assert (off <= tol).all(), (i, j, "lse", (off / tol).max().item())


HEADS = [(4, 2), (8, 8), (32, 8), (7, 1), (24, 1), (66, 2)]


@pytest.mark.parametrize("kv,qt", [(BF, BF), (HF, HF), (E4, BF), (E4, HF)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("t", [1, 3])
@pytest.mark.parametrize("hq,hkv", HEADS)
def test_types_heads_and_lengths(kv, qt, d, t, hq, hkv):
    lens = [0, 1, 2, 15, 16, 17, 63, 64, 65, 129, 400]
    page = {1: 16, 2: 32, 8: 64}[hkv]
    c, slots, _ = build(lens, [], [], page=page, hkv=hkv, d=d, dtype=kv, seed=hq + d + t)
    q = queries(len(lens), hq, t, d, qt, hq)
    out, lse = c.attend(q, ints(slots))
    c.check_status()
    compare(c, q, out, lse, slots)


@pytest.mark.parametrize("t", [1, 2, 5, 16])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("kv,d,hq,hkv", [(BF, 128, 8, 2), (HF, 64, 12, 3), (E4, 128, 16, 2), (E4, 64, 5, 1)])
def test_groups_that_share_a_prefix(t, page, kv, d, hq, hkv):
    """Prefixes of any length (whole pages are shared), groups of one and of many, members whose newest tokens reach into
    the shared part, empty members, and an empty group."""
    shared = [7 * 128 + 16, 300, 0, 150, 64, 50]
    members = [9, 4, 3, 1, 0, 5]
    rng = random.Random(t * page + d)
    lens = []
    for m, s in zip(members, shared):
        lens += [s + rng.choice([max(t, 1), t + 1, t + 70, t + 300]) for _ in range(m)]
    lens[10] = 0  # a member of the second group that has ended
    if t > 1:
        lens[-1] = shared[-1] // page * page  # nothing but shared tokens: its first queries do not see all of them
        if lens[-1] == 0:
            lens[-1] = 1
    c, slots, offsets = build(lens, [s if s >= page else 0 for s in shared], members, page=page, hkv=hkv, d=d, dtype=kv, seed=page + t)
    qt = HF if kv == HF else BF
    q = queries(len(lens), hq, t, d, qt, t)
    told = [s // page * page for s in shared]
    out, lse = c.attend(q, ints(slots), group_offsets=ints(offsets), shared_lens=ints(told))
    c.check_status()
    compare(c, q, out, lse, slots)
    # told that nothing is shared, or less: the same attention
    for less in ([0] * 6, [x // 3 for x in told]):
        out2, lse2 = c.attend(q, ints(slots), group_offsets=ints(offsets), shared_lens=ints(less))
        compare(c, q, out2, lse2, slots)
    out3, lse3 = c.attend(q, ints(slots))
    compare(c, q, out3, lse3, slots)


@pytest.mark.parametrize("kv,qt,d,hq,hkv,t", [(BF, BF, 128, 32, 8, 1), (HF, HF, 128, 32, 8, 4), (E4, BF, 128, 32, 8, 1), (E4, HF, 64, 32, 8, 2), (BF, BF, 64, 28, 4, 3)])
def test_a_long_prefix_and_many_samples(kv, qt, d, hq, hkv, t):
    lens = [5003 + (i * 97) % 700 + t for i in range(40)]
    c, slots, offsets = build(lens, [5000], [40], page=16, hkv=hkv, d=d, dtype=kv, seed=2)
    q = queries(40, hq, t, d, qt, 3, amp=2.0)
    out, lse = c.attend(q, ints(slots), group_offsets=ints(offsets), shared_lens=ints([5000 // 16 * 16]))
    c.check_status()
    compare(c, q, out, lse, slots)
    again, lse_again = c.attend(q, ints(slots), group_offsets=ints(offsets), shared_lens=ints([5000 // 16 * 16]))
    assert torch.equal(out, again) and torch.equal(lse, lse_again)


@pytest.mark.parametrize("kv", [BF, E4])
def test_one_long_sequence(kv):
    c, slots, _ = build([70001], [], [], page=128, hkv=1, d=128, dtype=kv, seed=4)
    q = queries(1, 8, 1, 128, BF, 5)
    out, lse = c.attend(q, ints(slots))
    compare(c, q, out, lse, slots)


@pytest.mark.parametrize("kv,qt", [(BF, BF), (HF, HF), (E4, BF)])
def test_large_scores_keep_their_precision(kv, qt):
    """Maxima that grow along the keys, so that accumulators are scaled again and again; scores of some hundreds."""
    lens = [700, 90]
    c, slots, offsets = build(lens, [64], [2], hkv=2, d=64, dtype=kv, seed=6)
    table = c.page_table[slots[0], :44].long()
    order = torch.ones(c.k.shape[1], device=DEV)
    order[table] = torch.linspace(0.1, 6.0, 44, device=DEV)
    c.k.copy_((c.k.float() * order[None, :, None, None, None]).to(c.k.dtype))
    q = queries(2, 8, 1, 64, qt, 7, amp=4.0)
    for args in ({}, dict(group_offsets=ints(offsets), shared_lens=ints([64]))):
        out, lse = c.attend(q, ints(slots), **args)
        compare(c, q, out, lse, slots)


@pytest.mark.parametrize("amp", [2.0 ** -100, 2.0 ** 60])
def test_queries_of_any_magnitude_over_an_e4m3_cache(amp):
    """bf16 queries beyond the range of f16: the power of two per row keeps them exact."""
    c, slots, _ = build([130, 77], [], [], hkv=2, d=128, dtype=E4, seed=8)
    q = (queries(2, 4, 1, 128, BF, 9).float() * amp).to(BF)
    q[0, 0] = 0
    out, lse = c.attend(q, ints(slots), softmax_scale=1.0 / amp / 16)
    compare(c, q, out, lse, slots, scale=1.0 / amp / 16)


def test_padding_rows_and_rows_behind_the_last_group():
    lens = [40, 100, 77, 30, 64]
    c, slots, offsets = build(lens, [32, 32], [2, 2], hkv=2, d=64, seed=10)
    q = queries(8, 4, 2, 64, BF, 11)
    named = [slots[0], slots[1], -1, slots[2], slots[3], 10 ** 9, slots[4], -1]
    out = torch.full((8, 4, 2, 64), 7.0, dtype=BF, device=DEV)
    got, lse = c.attend(q, ints(named), group_offsets=ints([0, 3, 6]), shared_lens=ints([32, 32]), out=out)
    c.check_status()
    assert got is out
    compare(c, q, out, lse, named, rows=range(6))
    assert (out[6:] == 7.0).all()


@pytest.mark.parametrize("offsets", [[0, 3, 2], [-1, 2, 4], [0, 2, 5]])
def test_offsets_that_are_none_are_reported_and_nothing_is_written(offsets):
    c, slots, _ = build([40, 100, 77, 30], [32, 32], [2, 2], hkv=2, d=64, seed=10)
    q = queries(4, 4, 1, 64, BF, 11)
    out = torch.full((4, 4, 1, 64), 7.0, dtype=BF, device=DEV)
    c.attend(q, ints(slots), group_offsets=ints(offsets), shared_lens=ints([32, 32]), out=out)
    with pytest.raises(ValueError, match="offsets"):
        c.check_status()
    assert (out == 7.0).all()
    c.check_status()


@pytest.mark.parametrize("kv", [BF, HF, E4])
@pytest.mark.parametrize("page", [16, 64])
def test_pages_that_the_table_does_not_name_hold_no_keys(kv, page):
    lens = [200, 333, 10]
    c, slots, _ = build(lens, [], [], page=page, hkv=2, d=64, dtype=kv, seed=12)
    holes = []
    for row, at, what in ((0, 1, -1), (1, 0, c.k.shape[1]), (1, 3, 2 ** 30), (2, 0, -5)):
        c.page_table[slots[row], at] = what
        holes += [(row, x) for x in range(at * page, min(lens[row], (at + 1) * page))]
    q = queries(3, 6, 1, 64, HF if kv == HF else BF, 13)
    out, lse = c.attend(q, ints(slots))
    c.check_status()
    compare(c, q, out, lse, slots, holes=holes)


@pytest.mark.parametrize("kv", [BF, HF, E4])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_drafted_token_does_not_reach_the_queries_before_it(kv, bad):
    t, lens = 4, [70, 64, 129, 5]
    c, slots, _ = build(lens, [], [], hkv=2, d=128, dtype=kv, seed=14)
    q = queries(4, 8, t, 128, HF if kv == HF else BF, 15)
    clean, clean_lse = c.attend(q, ints(slots))
    compare(c, q, clean, clean_lse, slots)
    for i, s in enumerate(slots):
        pos = lens[i] - 2  # seen by queries 2 and 3
        p = int(c.page_table[s, pos // 16])
        if kv == E4:
            c.v.view(torch.uint8)[0, p, :, pos % 16] = 0x7f
            c.k.view(torch.uint8)[0, p, :, pos % 16] = 0x7f
        else:
            c.v[0, p, :, pos % 16] = bad
            c.k[0, p, :, pos % 16] = float("nan")
    out, lse = c.attend(q, ints(slots))
    assert torch.equal(out[:, :, :2], clean[:, :, :2]) and torch.equal(lse[:, :, :2], clean_lse[:, :, :2])
    assert out[:, :, 2:].isnan().all()


def test_strides_layers_and_the_softmax_scale():
    lens = [37, 290, 64]
    c, slots, offsets = build(lens, [32], [3], hkv=2, d=64, layers=3, seed=16)
    wide = torch.randn(3, 2, 8 * 64 + 128, generator=torch.Generator().manual_seed(1)).to(BF).to(DEV)  # [n, T, ...]: a projection's rows
    q = wide[:, :, 64:64 + 512].view(3, 2, 8, 64).transpose(1, 2)
    for layer in range(3):
        buf = torch.zeros(3, 2, 8, 64, dtype=BF, device=DEV)
        out, lse = c.attend(q, ints(slots), layer=layer, softmax_scale=0.3, out=buf.transpose(1, 2), group_offsets=ints(offsets), shared_lens=ints([32]))
        assert out.data_ptr() == buf.data_ptr()
        compare(c, q, out, lse, slots, layer=layer, scale=0.3)


def test_no_rows_and_slots_in_order():
    c, slots, _ = build([50, 0, 33], [], [], hkv=1, d=64, seed=17, shuffle_slots=False)
    out, lse = c.attend(queries(0, 4, 1, 64, BF, 0))
    assert out.shape == (0, 4, 1, 64) and lse.shape == (0, 4, 1)
    q = queries(3, 4, 1, 64, BF, 1)
    out, lse = c.attend(q)
    compare(c, q, out, lse, slots)


def test_a_large_batch():
    rng = random.Random(5)
    lens = [rng.choice([0, 1, 30, 100, 200]) for _ in range(2500)]
    c, slots, _ = build(lens, [], [], hkv=1, d=64, seed=18)
    q = queries(2500, 2, 1, 64, BF, 19)
    members = [1000, 500, 300, 700]
    out, lse = c.attend(q, ints(slots), group_offsets=ints([0, 1000, 1500, 1800, 2500]), shared_lens=ints([0, 0, 0, 0]))
    c.check_status()
    compare(c, q, out, lse, slots, rows=range(0, 2500, 7))


def test_what_is_refused():
    c, slots, _ = build([50, 20], [], [], hkv=2, d=64, seed=20)
    q = queries(2, 4, 1, 64, BF, 0)
    s = ints(slots)
    with pytest.raises(ValueError, match="multiple of Hkv"):
        c.attend(queries(2, 5, 1, 64, BF, 0), s)
    with pytest.raises(ValueError, match="T=17"):
        c.attend(queries(2, 4, 17, 64, BF, 0), s)
    with pytest.raises(ValueError, match="\\[n, Hq, T, 64\\]"):
        c.attend(queries(2, 4, 1, 128, BF, 0), s)
    with pytest.raises(TypeError, match="the cache"):
        c.attend(q.half(), s)
    with pytest.raises(ValueError, match="entries"):
        c.attend(q, ints([0]))
    with pytest.raises(TypeError, match="int32"):
        c.attend(q, s.long())
    with pytest.raises(ValueError, match="go together"):
        c.attend(q, s, group_offsets=ints([0, 2]))
    with pytest.raises(ValueError, match="must have 2 entries"):
        c.attend(q, s, group_offsets=ints([0, 2, 2]), shared_lens=ints([0]))
    with pytest.raises(ValueError, match="groups=3"):
        c.attend(q, s, group_offsets=ints([0, 1, 2, 2]), shared_lens=ints([0, 0, 0]))
    with pytest.raises(ValueError, match="layer 1 of 1"):
        c.attend(q, s, layer=1)
    with pytest.raises(ValueError, match="alignment"):
        c.attend(torch.zeros(2 * 4 * 64 + 1, dtype=BF, device=DEV)[1:].view(2, 4, 1, 64), s)
    with pytest.raises(ValueError, match="out must"):
        c.attend(q, s, out=torch.zeros(2, 4, 1, 64, dtype=HF, device=DEV))
    with pytest.raises(RuntimeError, match="must live"):
        c.attend(q.cpu(), s)
    c.check_status()


def test_two_captured_steps_are_replayed_in_any_order_with_eager_calls_between():
    lens = [150, 170, 160]
    c, slots, offsets = build(lens, [128], [3], hkv=2, d=128, seed=21, width=40, spare_pages=60)
    s, off, sh = ints(slots), ints(offsets), ints([128])
    qs = [queries(3, 8, 1, 128, BF, 30), queries(3, 8, 2, 128, BF, 31)]
    graphs, results = [], []
    side = torch.cuda.Stream()
    for q in qs:
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                results.append(c.attend(q, s, group_offsets=off, shared_lens=sh))
        torch.cuda.current_stream().wait_stream(side)
        graphs.append(g)
    for turn in range(4):
        for which in ((0, 1), (1, 0))[turn % 2]:
            qs[which].normal_()
            graphs[which].replay()
            eager = c.attend(qs[1 - which], s)
            compare(c, qs[which], *results[which], slots)
            compare(c, qs[1 - which], *eager, slots)
        c.extend(s, ints([3, 40, 17]))  # the lengths are read by the replay
        c.k.nan_to_num_(nan=0.25), c.v.nan_to_num_(nan=-0.5)
    c.check_status()


def test_a_generation_from_the_prompt_to_compaction():
    """What a serving program does: prompts in, samples forked, tokens drafted and attended to, losers freed, the pool
    compacted, and on; against a dense history kept in 64 bits."""
    rng = random.Random(3)
    hkv, hq, d, page = 2, 8, 64, 16
    c = PagedKVCache.empty(200, page, hkv, d, 20, 30, dtype=BF, n_layers=2, device=DEV)
    history = {}  # slot -> [(k, v) of each layer], [tokens, hkv, d]
    gen = torch.Generator().manual_seed(1)

    def fresh(n, t):
        return [torch.randn(n, hkv, t, d, generator=gen).to(BF).to(DEV) for _ in range(2)]

    def grow(slots, t):
        c.extend(ints(slots), ints([t] * len(slots)))
        for layer in range(2):
            k, v = fresh(len(slots), t)
            c.write(k, v, ints(slots), layer=layer)
            for i, s in enumerate(slots):
                for which, x in enumerate((k, v)):
                    old = history.setdefault(s, [[None, None], [None, None]])[layer][which]
                    new = x[i].transpose(0, 1)
                    history[s][layer][which] = new if old is None else torch.cat([old, new])

    def look(slots, t, **args):
        q = queries(len(slots), hq, t, d, BF, rng.randrange(10 ** 6))
        for layer in range(2):
            out, lse = c.attend(q, ints(slots), layer=layer, **args)
            for i, s in enumerate(slots):
                k, v = (x.double().repeat_interleave(hq // hkv, 1) for x in history[s][layer])
                for j in range(t):
                    m = len(k) - (t - 1 - j)
                    z = torch.einsum("hd,khd->hk", q[i, :, j].double(), k[:m]) * d ** -0.5
                    w = torch.softmax(z, -1)
                    want = torch.einsum("hk,khd->hd", w, v[:m])
                    a = torch.einsum("hk,khd->hd", w, v[:m].abs())
                    e = 2.0 ** -19 * d ** -0.5 * torch.einsum("hd,khd->hk", q[i, :, j].double().abs(), k[:m].abs()).amax()
                    tol = a * (2.0 ** -8 + 2 * e + 2.0 ** -17) + want.abs() * 2.0 ** -8 + 2.0 ** -20
                    assert ((out[i, :, j].double() - want).abs() <= tol).all(), (s, j)
                    assert ((lse[i, :, j].double() - torch.logsumexp(z, -1)).abs() <= e + 2.0 ** -17).all()

    grow([0], 100), grow([1], 47)
    look([1, 0], 1)
    children = {0: [2, 3, 4, 5, 6], 1: [7, 8]}
    for parent, kids in children.items():
        c.fork(ints([parent] * len(kids)), ints(kids))
        for s in kids:
            history[s] = [[x.clone() for x in layer] for layer in history[parent]]
    order = [0, 2, 3, 4, 5, 6, 1, 7, 8]
    groups = dict(group_offsets=ints([0, 6, 9]), shared_lens=ints([96, 32]))
    for step in range(12):
        t = rng.choice([1, 1, 3])
        grow(order, t)
        look(order, t, **groups)
        if step == 5:
            c.free(ints([3, 8]))
            del history[3], history[8]
            c.compact()
            order = [0, 2, 4, 5, 6, 1, 7]
            groups["group_offsets"] = ints([0, 5, 7])
            look(order, t, **groups)
    c.fork(ints([4]), ints([8]))
    history[8] = [[x.clone() for x in layer] for layer in history[4]]
    grow([8, 4], 20)
    look([8, 4, 7], 2)
    c.check_status()
    c.free(ints(list(range(20))))
    c.compact()
    assert int(c.ref_counts.sum()) == 0 and int(c.seq_lens.sum()) == 0 and (c.page_table == -1).all()
    c.check_status()


def test_pools_and_tables_that_are_views():
    """K and V as views of one tensor with layers between them, a table whose rows are part of a wider tensor."""
    layers, pages, page, hkv, d = 3, 30, 32, 2, 128
    gen = torch.Generator().manual_seed(40)
    both = torch.randn(layers, pages, 2, hkv, page, d, generator=gen).to(BF).to(DEV)
    wide = torch.full((4, 40), 7777, dtype=torch.int32, device=DEV)
    table = wide[:, 5:17]
    c = PagedKVCache(both[:, :, 0], both[:, :, 1], table, torch.zeros(4, dtype=torch.int32, device=DEV), torch.zeros(pages, dtype=torch.int32, device=DEV))
    table.fill_(-1)
    slots = [2, 0, 3]
    c.extend(ints(slots), ints([300, 33, 200]))
    c.fork(ints([2]), ints([1]))
    assert (wide[:, :5] == 7777).all() and (wide[:, 17:] == 7777).all()
    q = queries(4, 6, 2, d, BF, 41)
    for layer in range(layers):
        out, lse = c.attend(q, ints([2, 1, 0, 3]), layer=layer, group_offsets=ints([0, 2, 4]), shared_lens=ints([288, 0]))
        compare(c, q, out, lse, [2, 1, 0, 3], layer=layer)
    c.check_status()


def test_a_pool_beyond_32_bit_offsets():
    """Pages whose elements lie beyond 2^32: written, copied, forked, attended to (both kinds of units)."""
    page, hkv, d, pages = 128, 8, 128, 33500  # 4.4e9 elements a pool
    k, v = [torch.empty(1, pages, hkv, page, d, dtype=BF, device=DEV) for _ in range(2)]
    refs = torch.ones(pages, dtype=torch.int32, device=DEV)
    refs[pages - 40:] = 0
    refs[3] = 0
    c = PagedKVCache(k, v, torch.full((8, 20), -1, dtype=torch.int32, device=DEV), torch.zeros(8, dtype=torch.int32, device=DEV), refs)
    c.extend(ints([0, 1]), ints([300, 700]))
    for s, n in ((0, 300), (1, 700)):
        gen = torch.Generator().manual_seed(s)
        c.write(*[torch.randn(1, hkv, n, d, generator=gen).to(BF).to(DEV) for _ in range(2)], ints([s]))
    c.fork(ints([1, 1, 1]), ints([2, 3, 4]))
    assert int(c.page_table[1, 0]) == pages - 38 and int(c.page_table[0, 0]) == 3
    q = queries(5, 16, 1, d, BF, 42)
    for args in ({}, dict(group_offsets=ints([0, 1, 5]), shared_lens=ints([0, 640]))):
        out, lse = c.attend(q, ints([0, 1, 2, 3, 4]), **args)
        compare(c, q, out, lse, [0, 1, 2, 3, 4])
    last = int(c.page_table[1, 1])
    c.copy_pages(ints([last]), ints([pages - 1]))
    assert torch.equal(c.k[0, pages - 1], c.k[0, last]) and torch.equal(c.v[0, pages - 1], c.v[0, last])
    c.free(ints([0]))
    c.compact()  # the last of the used pages moves into the hole
    out2, lse2 = c.attend(q[1:], ints([1, 2, 3, 4]))
    assert torch.equal(out2, c.attend(q[1:], ints([1, 2, 3, 4]))[0])
    compare(c, q[1:], out2, lse2, [1, 2, 3, 4])
    c.check_status()


@pytest.mark.parametrize("hq,hkv,t", [(128, 1, 16), (64, 2, 16), (40, 8, 3)])
def test_many_rows_of_one_sequence(hq, hkv, t):
    lens = [500, 17, 260]
    c, slots, _ = build(lens, [], [], hkv=hkv, d=64, seed=43)
    q = queries(3, hq, t, 64, BF, 44)
    out, lse = c.attend(q, ints(slots))
    compare(c, q, out, lse, slots)
    lens = [400, 300, 271 + t]
    c, slots, offsets = build(lens, [256], [3], hkv=hkv, d=64, seed=45)
    out, lse = c.attend(q, ints(slots), group_offsets=ints(offsets), shared_lens=ints([256]))
    compare(c, q, out, lse, slots)
    c.check_status()


def test_thousands_of_groups():
    n = 4096
    lens = [40 + i % 30 for i in range(n)]
    members = [2] * (n // 2)
    c, slots, offsets = build(lens, [32] * len(members), members, hkv=1, d=64, seed=46)
    q = queries(n, 4, 1, 64, BF, 47)
    out, lse = c.attend(q, ints(slots), group_offsets=ints(offsets), shared_lens=ints([32] * len(members)))
    c.check_status()
    compare(c, q, out, lse, slots, rows=list(range(0, n, 61)) + [n - 1])
    ones = ints(list(range(n + 1)))
    out, lse = c.attend(q, ints(slots), group_offsets=ones, shared_lens=ints([32] * n))
    compare(c, q, out, lse, slots, rows=range(0, n, 97))


@pytest.mark.parametrize("qt", [BF, HF])
def test_scales_of_either_sign_and_zero(qt):
    lens = [200 + 16, 200 + 33, 200 + 7]
    c, slots, offsets = build(lens, [192], [3], hkv=3, d=128, dtype=E4, seed=48)
    c.k_scale[0] = torch.tensor([0.1, -0.13, 0.0], device=DEV)
    c.v_scale[0] = torch.tensor([-0.2, 0.1, 0.3], device=DEV)
    q = queries(3, 12, 1, 128, qt, 49)
    for args in ({}, dict(group_offsets=ints(offsets), shared_lens=ints([192]))):
        out, lse = c.attend(q, ints(slots), **args)
        compare(c, q, out, lse, slots)


def test_what_is_no_number_shows_in_its_row_alone():
    lens = [300, 280, 290]
    c, slots, offsets = build(lens, [256], [3], hkv=2, d=128, seed=50)
    q = queries(3, 8, 1, 128, BF, 51)
    args = dict(group_offsets=ints(offsets), shared_lens=ints([256]))
    clean, clean_lse = c.attend(q, ints(slots), **args)
    bad = q.clone()
    bad[1, 2, 0, 5] = float("nan")
    out, lse = c.attend(bad, ints(slots), **args)
    assert out[1, 2].isnan().all() and lse[1, 2].isnan().all()
    keep = torch.ones(3, 8, dtype=torch.bool)
    keep[1, 2] = False
    assert torch.equal(out[keep.to(DEV)], clean[keep.to(DEV)]) and torch.equal(lse[keep.to(DEV)], clean_lse[keep.to(DEV)])
    # a shared key that is no number: every row of its kv head, and none of the other's
    p = int(c.page_table[slots[0], 3])
    c.k[0, p, 1, 7] = float("nan")
    out, lse = c.attend(q, ints(slots), **args)
    assert out[:, 4:].isnan().all() and torch.equal(out[:, :4], clean[:, :4])


def test_calls_on_two_streams_at_once():
    lens = [900 + 40 * i for i in range(12)]
    c, slots, offsets = build(lens, [800], [12], hkv=2, d=128, seed=52)
    qs = [queries(12, 8, t, 128, BF, 53 + t) for t in (1, 2)]
    args = dict(group_offsets=ints(offsets), shared_lens=ints([800]))
    s = ints(slots)
    want = [c.attend(q, s, **args) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    got = [[], []]
    for turn in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(c.attend(qs[i], s, **args))
    torch.cuda.synchronize()
    for i in range(2):
        for out, lse in got[i]:
            assert torch.equal(out, want[i][0]) and torch.equal(lse, want[i][1])
    c.check_status()


@pytest.mark.parametrize("length", [-5, 2 ** 31 - 1])
def test_lengths_that_cannot_be_are_cut_to_the_table(length):
    c, slots, _ = build([64, 64], [], [], hkv=1, d=64, width=4, seed=54)
    q = queries(2, 4, 1, 64, BF, 55)
    c.seq_lens[slots[1]] = length
    out, lse = c.attend(q, ints(slots))
    c.check_status()
    c.seq_lens[slots[1]] = 64 if length > 0 else 0
    compare(c, q, out, lse, slots)


@pytest.mark.parametrize("scale", [-0.1, float("nan"), float("inf")])
def test_a_softmax_scale_that_cannot_be_is_refused(scale):
    c, slots, _ = build([50, 20], [], [], hkv=2, d=64, seed=20)
    with pytest.raises(ValueError, match="softmax_scale"):
        c.attend(queries(2, 4, 1, 64, BF, 0), ints(slots), softmax_scale=scale)


def test_an_empty_list_of_groups_is_refused():
    """Rows in no group are left as they were, which with no group at all is every row; a C call with groups == 0 computes all of them."""
    c, slots, _ = build([50, 20], [], [], hkv=2, d=64, seed=20)
    with pytest.raises(ValueError, match="no groups"):
        c.attend(queries(2, 4, 1, 64, BF, 0), ints(slots), group_offsets=ints([0]), shared_lens=ints([]))
    out, lse = c.attend(queries(0, 4, 1, 64, BF, 0), ints([]), group_offsets=ints([0]), shared_lens=ints([]))
    assert out.shape == (0, 4, 1, 64) and lse.shape == (0, 4, 1)


@pytest.mark.parametrize("d,page,dtype", [(128, 16, BF), (64, 128, E4)])
@pytest.mark.parametrize("n,t", [(1, 1), (2, 4), (31, 1), (32, 2), (32, 4), (33, 2), (64, 1)])
def test_rows_without_groups_around_the_size_that_needs_no_plan(n, t, d, page, dtype):
    """One row, several, and both sides of 32 rows; lengths of zero, one and many, padding in the middle, a long row beside short ones."""
    rng = random.Random(n * 10 + t)
    lens = [rng.choice([0, 1, t, 15, 16, 17, 130, 700]) for _ in range(n)]
    lens[n // 2] = 5000
    c, slots, _ = build(lens, [], [], hkv=2, d=d, page=page, dtype=dtype, seed=n)
    named = list(slots)
    if n > 2:
        named[1], named[n - 1] = -1, 10 ** 9
        named[0] = named[n // 2]  # the same sequence twice
    q = queries(n, 8, t, d, BF, n)
    out, lse = c.attend(q, ints(named))
    c.check_status()
    compare(c, q, out, lse, named)
    for _ in range(3):  # cold or warm, early or late: the same bits
        again, lse2 = c.attend(q, ints(named))
        assert torch.equal(again, out) and torch.equal(lse2, lse)


def test_calls_that_differ_follow_one_another_without_a_pause():
    """Lengths, tables, groups, tokens and the kind of call change from one to the next on one stream, in the same workspace memory: each
    call sees its own plan, and not what one before it left."""
    lens = [700, 690, 1500, 333, 1481, 64, 900, 910]
    c, slots, _ = build(lens, [640, 320], [2, 2], hkv=2, d=128, seed=60)
    table, seq = c.page_table.clone(), c.seq_lens.clone()
    c.k.nan_to_num_(nan=0.25), c.v.nan_to_num_(nan=-0.5)
    turned = table.clone()
    turned[slots[6]], turned[slots[7]] = table[slots[7]], table[slots[6]]  # as many pages
    states = [(table, seq), (turned, (seq - 130).clamp(min=0)), (table, (seq // 3)), (turned, (seq - 17).clamp(min=0))]
    kinds = [dict(group_offsets=ints([0, 2, 4, 8]), shared_lens=ints([640, 320, 0])), {}, dict(group_offsets=ints([0, 2, 8]), shared_lens=ints([208, 0])),
             dict(group_offsets=ints([0, 1, 2, 8]), shared_lens=ints([640, 640, 0]))]
    qs = [queries(8, 8, t, 128, BF, 61 + t) for t in (1, 2, 4)]
    rng = random.Random(6)
    order = [(rng.randrange(4), rng.randrange(4), rng.randrange(3)) for _ in range(60)]
    s, results = ints(slots), []
    torch.cuda.synchronize()
    for state, kind, which in order:
        c.page_table.copy_(states[state][0]), c.seq_lens.copy_(states[state][1])
        results.append(c.attend(qs[which], s, **kinds[kind]))
        results[-1] += c.attend(qs[which], s, **kinds[kind - 1])
    c.check_status()
    for (state, kind, which), (out, lse, out2, lse2) in zip(order, results):
        c.page_table.copy_(states[state][0]), c.seq_lens.copy_(states[state][1])
        compare(c, qs[which], out, lse, slots)
        compare(c, qs[which], out2, lse2, slots)


@pytest.mark.parametrize("n,groups", [(3071, 0), (3008, 0), (2000, 714)])
def test_calls_whose_plan_takes_just_under_48_kb_of_shared_memory(n, groups):
    """In a process of their own: a larger call before them would have asked for more."""
    import pathlib
    import subprocess
    import sys

    text = f"""
import test_attn_paged_gpu as A, test_kv_cache_gpu as K
n, groups = {n}, {groups}
lens = [20 + i % 7 for i in range(n)]
members = [2] * groups
c, slots, offsets = A.build(lens, [16] * groups, members, hkv=1, d=64, seed=70)
q = A.queries(n, 2, 1, 64, A.BF, 71)
more = dict(group_offsets=A.ints(offsets), shared_lens=A.ints([16] * groups)) if groups else {{}}
out, lse = c.attend(q, A.ints(slots), **more)
c.check_status()
A.compare(c, q, out, lse, slots, rows=range(0, 2 * groups or n, 101))
seqs = list(range(262144 - 4090, 262144))
c = K.make(pages=4096, heads=1, layers=1, seqs=262144, width=1)
c.extend(K.ints(seqs), K.ints([3] * 4090))
c.check_status()
assert int(c.seq_lens.sum()) == 3 * 4090 and (c.page_table[seqs, 0] == K.ints(list(range(4090)))).all()
"""
    root = pathlib.Path(__file__).resolve().parents[1]
    done = subprocess.run([sys.executable, "-c", text], cwd=root, capture_output=True, text=True, timeout=240,
                          env={**__import__("os").environ, "PYTHONPATH": f"{root / 'fp4-fa4_b200'}:{root / 'tests'}:{root / 'oracle'}"})
    assert done.returncode == 0, done.stderr[-2000:]


@pytest.mark.parametrize("scale", [0.0, -0.0, 0, 1e-46, 1e39, -1e39, -float("inf")])
def test_a_softmax_scale_that_is_no_positive_number_in_32_bits_is_refused(scale):
    """Zero is no word for the default: None is."""
    c, slots, _ = build([50, 20], [], [], hkv=2, d=64, seed=20)
    with pytest.raises(ValueError, match="softmax_scale"):
        c.attend(queries(2, 4, 1, 64, BF, 0), ints(slots), softmax_scale=scale)


def test_the_softmax_scale_may_be_any_positive_number():
    c, slots, _ = build([50, 20], [], [], hkv=2, d=64, seed=20)
    q = queries(2, 4, 1, 64, BF, 0)
    for scale in (1, 2.0 ** -100, 0.125, None):
        out, lse = c.attend(q, ints(slots), softmax_scale=scale)
        compare(c, q, out, lse, slots, scale=scale)


@pytest.mark.parametrize("d,kv", [(64, BF), (128, HF), (128, E4)])
@pytest.mark.parametrize("t", [1, 3])
@pytest.mark.parametrize("wrong", [False, True])
def test_rows_that_are_not_computed_are_no_memory_of_something_else(d, kv, t, wrong):
    """Rows in no group, and every row where the offsets are none: LSE -inf, and O 0 unless the caller brought it."""
    lens = [40, 100, 77, 30, 64, 50]
    c, slots, _ = build(lens, [32, 32], [2, 2], hkv=2, d=d, dtype=kv, seed=80)
    qt = BF if kv == E4 else kv
    q = queries(6, 4, t, d, qt, 81)
    offsets, rest = ([1, 3, 2], range(6)) if wrong else ([1, 2, 4], (0, 4, 5))
    args = dict(group_offsets=ints(offsets), shared_lens=ints([0, 0]))
    for mine in (None, torch.full_like(q, 7.0)):
        junk = [torch.full((6, 4, t, d), float("nan"), dtype=qt, device=DEV), torch.full((6, 4, t), float("nan"), device=DEV)]
        del junk  # the next tensors of these sizes lie there
        out, lse = c.attend(q, ints(slots), out=mine, **args)
        for i in rest:
            assert (out[i] == (0.0 if mine is None else 7.0)).all() and (lse[i] == -math.inf).all()
        if not wrong:
            compare(c, q, out, lse, slots, rows=(1, 2, 3))
    if wrong:
        with pytest.raises(ValueError, match="offsets"):
            c.check_status()
    c.check_status()


def test_a_backward_pass_is_refused_and_not_left_out():
    lens = [50, 20]
    c, slots, _ = build(lens, [], [], hkv=2, d=64, seed=20)
    s = ints(slots)
    plain = queries(2, 4, 1, 64, BF, 0)
    want, want_lse = c.attend(plain, s)
    q = plain.clone().requires_grad_()
    buf = torch.zeros_like(plain)
    for given in (None, buf, buf):
        out, lse = c.attend(q * 1, s, out=given)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
        assert given is None or (out.data_ptr() == buf.data_ptr() and torch.equal(buf, want) and not buf.requires_grad)
        with pytest.raises(RuntimeError, match="no gradient"):
            out.float().sum().backward()
        with pytest.raises(RuntimeError, match="no gradient"):
            c.attend(q, s)[1].sum().backward()
    with torch.no_grad():
        out, lse = c.attend(q, s)
    assert not out.requires_grad and torch.equal(out, want)
    assert not want.requires_grad and q.grad is None


def test_findings_of_the_pages_and_of_the_attention_are_both_told():
    c, slots, _ = build([40, 100], [], [], hkv=2, d=64, seed=10)
    q = queries(2, 4, 1, 64, BF, 11)
    for _ in range(2):
        c.extend(ints(slots), ints([1, -1]))
        c.attend(q, ints(slots), group_offsets=ints([0, 3]), shared_lens=ints([0]))
        for text in ("negative", "offsets of 1 groups"):
            with pytest.raises(ValueError, match=text):
                c.check_status()
        c.check_status()


def test_a_first_call_may_be_a_captured_one():
    """A process whose first extend, write and attend are captured, and replayed with lengths that grow."""
    import os
    import pathlib
    import subprocess
    import sys

    text = """
import torch, test_attn_paged_gpu as A
from fa4b import PagedKVCache
c, slots, offsets = A.build([150, 170, 160], [128], [3], hkv=2, d=128, seed=21, width=40, spare_pages=60)
s, one, off, sh = A.ints(slots), A.ints([1, 1, 1]), A.ints(offsets), A.ints([128])
q, k, v = A.queries(3, 8, 1, 128, A.BF, 30), A.queries(3, 2, 1, 128, A.BF, 31), A.queries(3, 2, 1, 128, A.BF, 32)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    c.extend(s, one)
    c.write(k, v, s)
    grouped = c.attend(q, s, group_offsets=off, shared_lens=sh)
    alone = c.attend(q, s)
for _ in range(20):
    q.normal_(), k.normal_(), v.normal_()
    g.replay()
    A.compare(c, q, *grouped, slots)
    A.compare(c, q, *alone, slots)
c.check_status()
assert c.seq_lens[slots].tolist() == [170, 190, 180]
"""
    root = pathlib.Path(__file__).resolve().parents[1]
    done = subprocess.run([sys.executable, "-c", text], cwd=root, capture_output=True, text=True, timeout=240,
                          env={**os.environ, "PYTHONPATH": f"{root / 'fp4-fa4_b200'}:{root / 'tests'}:{root / 'oracle'}"})
    assert done.returncode == 0, done.stderr[-2000:]


@pytest.mark.parametrize("kv", [BF, E4])
@pytest.mark.parametrize("page,width", [(16, 33), (128, 5)])
def test_sequences_that_fill_their_row_of_the_table(kv, page, width):
    lens = [page * width, page * width - 1, page * (width - 1) + 1]
    c, slots, offsets = build(lens, [page * (width - 2)], [3], page=page, hkv=2, d=128, dtype=kv, seed=90, width=width)
    for t in (1, 5):
        for hq in (8, 64):
            q = queries(3, hq, t, 128, BF, 91)
            for args in ({}, dict(group_offsets=ints(offsets), shared_lens=ints([page * (width - 2)]))):
                out, lse = c.attend(q, ints(slots), **args)
                compare(c, q, out, lse, slots)
    c.check_status()
