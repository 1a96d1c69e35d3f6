"""Paged cache on the device against a model on lists: every byte of pools, tables, lengths and counts."""

import random

import pytest
import torch

from fa4b import PagedKVCache
from kv_model import ModelCache

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float8_e4m3fn]


def ints(x, dev=DEV):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def make(pages=40, page=16, heads=2, d=64, seqs=12, width=9, layers=2, dtype=torch.bfloat16, seed=0, joint=False, dev=DEV):
    """A cache whose pools hold noise; with `joint`, K and V are views of one tensor (other strides)."""
    gen = torch.Generator().manual_seed(seed)
    scales = {}
    if dtype == torch.float8_e4m3fn:
        scales = {n: (0.01 + 0.02 * torch.rand(layers, heads, generator=gen)).to(dev) for n in ("k_scale", "v_scale")}
    noise = torch.randn(layers, pages, 2, heads, page, d, generator=gen).to(dtype).to(dev)
    k, v = noise[:, :, 0], noise[:, :, 1]
    if not joint:
        k, v = k.contiguous(), v.contiguous()
    return PagedKVCache(k, v, torch.full((seqs, width), -1, dtype=torch.int32, device=dev), torch.zeros(seqs, dtype=torch.int32, device=dev),
                        torch.zeros(pages, dtype=torch.int32, device=dev), **scales)


def values(n, heads, t, d, dtype, seed, dev=DEV):
    gen = torch.Generator().manual_seed(seed)
    return [(3 * torch.randn(n, heads, t, d, generator=gen)).to(dtype).to(dev) for _ in range(2)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page,d,heads,joint", [(16, 64, 2, False), (32, 128, 3, True), (128, 64, 1, True), (64, 128, 8, False)])
def test_a_random_run_of_all_calls(dtype, page, d, heads, joint):
    rng = random.Random(page * 7 + d)
    c = make(pages=60, page=page, heads=heads, d=d, seqs=14, width=7, layers=2, dtype=dtype, seed=3, joint=joint)
    m = ModelCache(c)
    src = torch.float16 if dtype == torch.float16 else torch.bfloat16
    for step in range(40):
        what = rng.choice(["extend", "extend", "free", "fork", "fork", "compact", "copy"])
        slots = rng.sample(range(14), rng.randint(1, 6))
        if what == "extend":
            new = [rng.choice([0, 1, 1, page - 1, page, page + 1, 2 * page + 5]) for _ in slots]
            c.extend(ints(slots), ints(new))
            if m.extend(slots, new):
                t = max(new)
                layer = rng.randrange(2)
                k, v = values(len(slots), heads, max(t, 1), d, src, step)
                c.write(k, v, ints(slots), n_new=ints(new), layer=layer)
                m.write(k, v, slots, new, layer)
        elif what == "free":
            c.free(ints(slots))
            m.free(slots)
        elif what == "fork":
            full = [s for s in range(14) if m.lens[s]]
            empty = [s for s in range(14) if not m.lens[s]]
            if full and empty:
                children = rng.sample(empty, rng.randint(1, len(empty)))
                parents = [rng.choice(full) for _ in children]
                c.fork(ints(parents), ints(children))
                m.fork(parents, children)
        elif what == "compact":
            c.compact()
            m.compact()
        else:
            free = [p for p, r in enumerate(m.refs) if r == 0]
            used = [p for p, r in enumerate(m.refs) if r > 0]
            n = min(len(free), len(used), 5)
            a, b = rng.sample(used, n), rng.sample(free, n)
            c.copy_pages(ints(a), ints(b))
            m.copy_pages(a, b)
        m.check(c, f"step {step}: {what}")
        m.invariants()


def test_status_of_a_run_without_faults_is_clean():
    c = make()
    c.extend(ints([0, 3]), ints([17, 40]))
    c.fork(ints([0, 0, 3]), ints([1, 2, 4]))
    c.free(ints([0, 0, 5]))  # a slot named twice and an empty one
    c.compact()
    c.copy_pages(ints([0, -1]), ints([30, 31]))
    c.check_status()


@pytest.mark.parametrize("call,error,text", [
    (lambda c: c.extend(ints([1, 12]), ints([5, 5])), ValueError, "slot 12 of 12"),
    (lambda c: c.extend(ints([1, -1]), ints([5, 5])), ValueError, "slot -1"),
    (lambda c: c.extend(ints([1, 2, 1]), ints([5, 5, 5])), ValueError, "second time"),
    (lambda c: c.extend(ints([1, 2]), ints([5, -5])), ValueError, "negative"),
    (lambda c: c.extend(ints([1, 2]), ints([5, 9 * 16 + 1])), ValueError, "too few"),
    (lambda c: c.extend(ints([0]), ints([2 ** 31 - 1])), ValueError, "too few"),
    (lambda c: c.extend(ints([1, 2, 3, 4, 5]), ints([140, 140, 140, 140, 140])), RuntimeError, "45 pages were asked for, 36 are free"),
    (lambda c: c.fork(ints([0, 0]), ints([3, 3])), ValueError, "second time"),
    (lambda c: c.fork(ints([0]), ints([0])), ValueError, "not empty"),
    (lambda c: c.fork(ints([0, 5]), ints([5, 6])), ValueError, "second time"),
    (lambda c: c.fork(ints([12]), ints([5])), ValueError, "slot 12"),
    (lambda c: c.fork(ints([0]), ints([99])), ValueError, "slot"),
    (lambda c: c.free(ints([50])), ValueError, "slot 50"),
    (lambda c: c.copy_pages(ints([0]), ints([40])), ValueError, "page 40 of 40"),
    (lambda c: c.copy_pages(ints([0, 1]), ints([9, 9])), ValueError, "page 9"),
    (lambda c: c.copy_pages(ints([0, 9]), ints([9, 11])), ValueError, "another pair"),
    (lambda c: c.copy_pages(ints([3]), ints([3])), ValueError, "page 3"),
    (lambda c: c.write(*values(1, 2, 3, 64, torch.bfloat16, 0), ints([77])), ValueError, "slot 77"),
])
def test_what_is_wrong_changes_nothing_and_is_reported_once(call, error, text):
    c = make()
    c.extend(ints([0]), ints([50]))
    m = ModelCache(c)
    call(c)
    m.check(c)
    with pytest.raises(error, match=text):
        c.check_status()
    c.check_status()


def test_free_leaves_out_what_is_wrong_and_frees_the_rest():
    c = make()
    c.extend(ints([0, 1]), ints([50, 20]))
    m = ModelCache(c)
    c.free(ints([1, -7, 1]))
    m.free([1])
    m.check(c)
    with pytest.raises(ValueError, match="slot -7"):
        c.check_status()


@pytest.mark.parametrize("n", [3, 600])
def test_copies_that_collide_are_left_out(n):
    c = make(pages=2 * n + 9, heads=1, layers=1)
    m = ModelCache(c)
    src, dst = list(range(n)), list(range(n, 2 * n))
    dst[1] = dst[0]
    src[-1] = 2 * n + 5
    c.copy_pages(ints(src), ints(dst))
    m.copy_pages(src, dst)
    m.check(c)
    with pytest.raises(ValueError, match="another pair"):
        c.check_status()


@pytest.mark.parametrize("pages", [1, 15, 16, 17, 4095, 4097, 40001])
@pytest.mark.parametrize("share", [0.0, 0.02, 0.5, 0.97, 1.0])
def test_compaction_of_pools_of_any_size(pages, share):
    rng = random.Random(pages)
    c = make(pages=pages, heads=1, layers=1, seqs=7, width=pages)
    used = rng.sample(range(pages), int(pages * share))
    table, lens, refs = c.page_table.cpu(), c.seq_lens.cpu(), c.ref_counts.cpu()
    for i in range(7):
        mine = used[i::7]
        table[i, :len(mine)] = torch.tensor(mine, dtype=torch.int32)
        lens[i] = max(0, 16 * len(mine) - i)
        refs[mine] = 1
    c.page_table.copy_(table), c.seq_lens.copy_(lens), c.ref_counts.copy_(refs)
    m = ModelCache(c)
    for _ in range(2):  # the second time there is nothing left to do
        c.compact()
        m.compact()
        m.check(c)
        m.invariants()
    c.check_status()


def test_claims_reach_over_a_long_list_of_counts_and_take_the_last_page():
    c = make(pages=40000, heads=1, layers=1, d=64, seqs=3000, width=40000)
    refs = torch.ones(40000, dtype=torch.int32)
    spare = [5, 16383, 16384, 20001, 39998, 39999]
    refs[spare] = 0
    c.ref_counts.copy_(refs)
    c.extend(ints([2999, 7]), ints([16 * 4, 2 * 16 - 3]))
    assert c.page_table[2999, :4].tolist() == spare[:4] and c.page_table[7, :2].tolist() == spare[4:]
    c.check_status()
    c.extend(ints([8]), ints([1]))
    with pytest.raises(RuntimeError, match="1 pages were asked for, 0 are free"):
        c.check_status()


def test_a_list_of_thousands():
    c = make(pages=5000, heads=1, layers=1, seqs=4500, width=3)
    m = ModelCache(c)
    order = random.Random(1).sample(range(4500), 4096)
    new = [1 + i % 17 for i in range(4096)]
    c.extend(ints(order[:2500]), ints(new[:2500]))
    assert m.extend(order[:2500], new[:2500])
    m.check(c)
    c.fork(ints(order[:1500]), ints(order[2500:4000]))
    assert m.fork(order[:1500], order[2500:4000])
    m.check(c)
    c.free(ints(order))
    m.free(order)
    m.check(c)
    c.check_status()
    with pytest.raises(ValueError, match="4096"):
        c.free(ints(list(range(4097))))


@pytest.mark.parametrize("scale", [2.0 ** -70, 1e-30, 1.9999998807907104, 2.0 ** 70, -0.037])
def test_an_e4m3_cache_with_an_odd_scale_stores_the_divisions_codes(scale):
    """Scales that the quotient by reciprocal does not cover, and values over the whole range: the 32-bit division's codes."""
    c = make(pages=30, heads=2, d=64, layers=1, dtype=torch.float8_e4m3fn)
    c.k_scale.fill_(scale), c.v_scale.fill_(0.0123)
    gen = torch.Generator().manual_seed(9)
    k, v = [(torch.randn(1, 2, 40, 64, generator=gen) * 10.0 ** torch.randint(-36, 36, (1, 2, 40, 64), generator=gen)).to(torch.bfloat16).to(DEV) for _ in range(2)]
    k[0, 0, 0, :4] = torch.tensor([float("inf"), -float("inf"), float("nan"), 0.0])
    v[0, 0, 0, :4] = k[0, 0, 0, :4]
    c.extend(ints([3]), ints([40]))
    m = ModelCache(c)
    c.write(k, v, ints([3]))
    m.write(k, v, [3], None, 0)
    m.check(c)


@pytest.mark.parametrize("src", [torch.bfloat16, torch.float16])
def test_what_an_e4m3_cache_stores(src):
    """Against the quotient in 64 bits: the 32-bit quotient is off by at most half a step (2^-24 relative), the code by half
    an E4M3 step of it (2^-4 relative, 2^-10 below 2^-6); clamped at 448, NaN kept."""
    c = make(pages=30, heads=3, d=128, layers=2, dtype=torch.float8_e4m3fn)
    k, v = values(2, 3, 37, 128, src, 5)
    k[0, 0, 0, :6] = torch.tensor([1e4, -1e4, float("inf"), -float("inf"), float("nan"), 0.0])
    v[1, 2, 5, :64] = torch.linspace(-1e-4, 1e-4, 64)
    c.extend(ints([4, 2]), ints([37, 37]))
    c.write(k, v, ints([4, 2]), layer=1)
    c.check_status()
    for i, s in enumerate([4, 2]):
        for pool, x, scale in ((c.k, k, c.k_scale), (c.v, v, c.v_scale)):
            rows = pool[1, c.page_table[s, :3].long()].float().permute(1, 0, 2, 3).flatten(1, 2)[:, :37].double()
            want = x[i].double() / scale[1].double()[:, None, None]
            assert torch.equal(rows.isnan(), want.isnan())
            want = want.clamp(-448, 448)
            tol = torch.maximum(want.abs() * 2 ** -4 * (1 + 2 ** -20), torch.full_like(want, 2 ** -10)) + want.abs() * 2 ** -24
            assert ((rows - want).abs() <= tol)[~want.isnan()].all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_write_takes_any_strides_and_leaves_other_tokens_alone(dtype):
    c = make(dtype=dtype, heads=4, d=64)
    src = torch.float16 if dtype == torch.float16 else torch.bfloat16
    c.extend(ints([1, 2, 3]), ints([20, 33, 7]))
    m = ModelCache(c)
    flat = torch.randn(3, 9, 3 * 4 * 64, dtype=torch.float32).to(src).to(DEV)  # [n, T, (q k v) heads x d], as a projection leaves it
    k, v = (flat[:, :, j * 256:(j + 1) * 256].view(3, 9, 4, 64).transpose(1, 2) for j in (1, 2))
    assert not k.is_contiguous()
    c.write(k, v, ints([1, 2, 3]), n_new=ints([9, 0, 12]), layer=0)  # 12 > T: the first 9 of 12; 12 > 7: positions below 0
    m.write(k, v, [1, 2, 3], [9, 0, 12], 0)
    m.check(c)
    c.write(k[:, :, :1], v[:, :, :1], ints([3, 1, 2]), layer=1)
    m.write(k[:, :, :1], v[:, :, :1], [3, 1, 2], None, 1)
    m.check(c)
    c.check_status()


def test_empty_lists_and_no_tokens():
    c = make()
    m = ModelCache(c)
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    c.free(none), c.extend(none, none), c.fork(none, none), c.copy_pages(none, none)
    c.write(*values(0, 2, 3, 64, torch.bfloat16, 0), none)
    c.write(*values(1, 2, 0, 64, torch.bfloat16, 0), ints([0]))
    c.compact()
    m.check(c)
    c.check_status()


def test_a_step_is_captured_and_replayed():
    c = make(pages=50, width=8)
    seqs, one = ints([0, 1]), ints([1, 1])
    c.extend(ints([0, 1, 2]), ints([14, 30, 33]))
    m = ModelCache(c)
    k, v = values(2, 2, 1, 64, torch.bfloat16, 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            c.extend(seqs, one)
            c.write(k, v, seqs)
            c.free(ints_static := torch.zeros(1, dtype=torch.int32, device=DEV) + 5)
            c.fork(seqs[:1], ints_static)
            c.compact()
    torch.cuda.current_stream().wait_stream(side)
    m.check(c)  # capturing ran nothing
    for step in range(5):
        k.normal_(), v.normal_()
        graph.replay()
        assert m.extend([0, 1], [1, 1])
        m.write(k, v, [0, 1], None, 0)
        m.free([5])
        assert m.fork([0], [5])
        m.compact()
        m.check(c, f"replay {step}")
        m.invariants()
    c.check_status()


def test_calls_follow_the_current_stream():
    c = make()
    side = torch.cuda.Stream()
    seqs, new = ints([0, 1]), ints([40, 16])
    m = ModelCache(c)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        c.extend(seqs, new)
        c.fork(ints([0]), ints([3]))
        c.check_status()
    m.extend([0, 1], [40, 16])
    m.fork([0], [3])
    m.check(c)


def full_pool(dtype=torch.bfloat16, length=48):
    """Slots 0 (forked into 3 at a page's end) and 1, each with `length` tokens written, and two pages left."""
    c = make(pages=8, dtype=dtype, layers=2)
    src = torch.float16 if dtype == torch.float16 else torch.bfloat16
    c.extend(ints([0, 1]), ints([length, length]))
    for layer in range(2):
        c.write(*values(2, 2, length, 64, src, layer), ints([0, 1]), layer=layer)
    c.fork(ints([0]), ints([3]))
    c.check_status()
    return c, src


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("seqs,new,error,text", [
    ([0, 1, 3], [1, 1, 1], RuntimeError, "3 pages were asked for, 2 are free"),
    ([3, 12, 1], [1, 1, 1], ValueError, "slot 12 of 12"),
    ([3, 1, 1], [2, 2, 2], ValueError, "second time"),
    ([1, 3], [9 * 16, 2], ValueError, "too few"),
    ([1, 0], [2, -2], ValueError, "negative"),
])
def test_a_write_behind_an_extend_that_was_refused_leaves_the_tokens_alone(dtype, seqs, new, error, text):
    """The step goes on (nothing synchronises): what is written then would land on the newest tokens, shared ones among them."""
    c, src = full_pool(dtype)
    m = ModelCache(c)
    c.extend(ints(seqs), ints(new))
    for layer in range(2):
        c.write(*values(len(seqs), 2, 2, 64, src, 7 + layer), ints(seqs), n_new=ints([2] * len(seqs)), layer=layer)
        c.write(*values(len(seqs), 2, 1, 64, src, 9 + layer), ints(seqs), layer=layer)
    m.check(c)
    with pytest.raises(error, match=text):
        c.check_status()
    c.write(*values(1, 2, 1, 64, src, 11), ints([seqs[0]]))  # the status says nothing about the slot's length: still no place
    m.check(c)
    with pytest.raises(ValueError, match=f"slot {seqs[0]}, whose last extend was refused"):
        c.check_status()
    c.check_status()


def test_slots_that_a_refused_extend_does_not_name_are_written_and_named_ones_again_after_the_next():
    c, src = full_pool()
    m = ModelCache(c)

    def write(seqs, seed, ok):
        k, v = values(len(seqs), 2, 2, 64, src, seed)
        c.write(k, v, ints(seqs))
        if ok:
            m.write(k, v, seqs, None, 0)
        m.check(c, str(seed))

    c.extend(ints([0, 3, 1]), ints([1, 1, 1]))  # three pages, two are free
    write([0, 3], 1, False)
    c.extend(ints([1]), ints([2]))  # another list, which fits
    assert m.extend([1], [2])
    write([1], 2, True)
    write([3], 3, False)
    c.extend(ints([3, 5]), ints([2, 0]))  # the last page
    assert m.extend([3, 5], [2, 0])
    write([3], 4, True)
    write([0], 5, False)
    c.free(ints([1]))  # gives pages back
    m.free([1])
    c.extend(ints([0]), ints([3]))
    assert m.extend([0], [3])
    write([0], 6, True)
    # a free and a fork open a slot as well
    c.extend(ints([7, 8]), ints([99, 99]))
    c.free(ints([8]))
    c.fork(ints([0]), ints([7]))
    m.free([8])
    assert m.fork([0], [7])
    write([7], 7, True)
    c.extend(ints([0]), ints([0]))
    write([0], 8, True)
    m.invariants()


def test_a_captured_step_is_replayed_through_a_full_pool():
    """Extend and write in one graph: replays that find too few pages change nothing, and the step works again once pages are there."""
    c, src = full_pool()
    seqs, new = ints([0, 1, 3]), ints([1, 1, 1])
    k, v = values(3, 2, 1, 64, src, 20)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            c.extend(seqs, new)
            c.write(k, v, seqs)
    torch.cuda.current_stream().wait_stream(side)
    m = ModelCache(c)
    for _ in range(2):
        k.normal_(), v.normal_()
        graph.replay()
        m.check(c)
    with pytest.raises(RuntimeError, match="3 pages were asked for"):
        c.check_status()
    c.free(ints([1]))
    m.free([1])
    for _ in range(3):
        k.normal_(), v.normal_()
        graph.replay()
        assert m.extend([0, 1, 3], [1, 1, 1])
        m.write(k, v, [0, 1, 3], None, 0)
        m.check(c)
    m.invariants()
    c.check_status()


@pytest.mark.parametrize("seqs", [12, 33, 4500])
def test_marks_of_refused_slots_are_a_slots_own(seqs):
    """First and last slots, neighbours in a word, and the other calls in between, which use the work area too."""
    c = make(pages=6000, heads=1, layers=1, seqs=seqs, width=1)
    named = sorted({0, 1, 9, seqs // 2, seqs - 2, seqs - 1})
    others = [s for s in range(seqs) if s not in named][:5]
    c.extend(ints(named + others), ints([7] * (len(named) + len(others))))
    c.extend(ints(named), ints([10] * len(named)))  # 17 tokens, rows of 16
    order = [s for s in range(seqs) if s not in named + others][: 2 * (seqs // 4)]
    half = len(order) // 2
    if half:
        c.extend(ints(order[:half]), ints([3] * half))
        c.fork(ints(order[:half]), ints(order[half:2 * half]))
        c.free(ints(order))
    c.copy_pages(ints(list(range(1200))), ints(list(range(3000, 4200))))
    c.compact()
    m = ModelCache(c)
    k, v = values(len(named) + len(others), 1, 2, 64, torch.bfloat16, 1)
    c.write(k, v, ints(named + others))
    m.write(k[len(named):], v[len(named):], others, None, 0)
    m.check(c)
    c.free(ints(named[:3]))
    m.free(named[:3])
    c.extend(ints(named), ints([1] * len(named)))
    assert m.extend(named, [1] * len(named))
    c.write(k[:len(named)], v[:len(named)], ints(named), n_new=ints([1] * len(named)))
    m.write(k[:len(named)], v[:len(named)], named, [1] * len(named), 0)
    m.check(c)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [16, 64])
def test_tokens_in_pages_that_several_slots_hold_are_not_written(dtype, page):
    """A write that reaches behind a fork: the tail is a slot's own, the pages before it belong to the samples too."""
    c = make(pages=40, page=page, heads=2, dtype=dtype)
    src = torch.float16 if dtype == torch.float16 else torch.bfloat16
    length = 5 * page + 7
    c.extend(ints([0]), ints([length]))
    c.fork(ints([0]), ints([4]))
    m = ModelCache(c)
    k, v = values(2, 2, length, 64, src, 1)
    c.write(k, v, ints([4, 0]), layer=1)
    own = [7, 7]
    m.write(k[:, :, -7:], v[:, :, -7:], [4, 0], own, 1)
    m.check(c)
    with pytest.raises(ValueError, match="entry [01] writes to page [0-4], which several slots hold"):
        c.check_status()
    c.free(ints([0]))  # then the pages are slot 4's alone
    m.free([0])
    c.write(k, v, ints([4, 4]), n_new=ints([length, 0]), layer=0)
    m.write(k, v, [4, 4], [length, 0], 0)
    m.check(c)
    c.check_status()


@pytest.mark.parametrize("n", [1024, 1025, 1030, 4096])
def test_collisions_in_long_lists_are_left_out(n):
    """Up to 1024 pairs are checked by the CTAs that copy, more by a launch before them: collisions and bad pages in its first and last warp."""
    c = make(pages=2 * n + 9, heads=1, layers=2)
    m = ModelCache(c)
    rng = random.Random(n)
    order = rng.sample(range(2 * n), 2 * n)
    src, dst = order[:n], order[n:]
    dst[1] = dst[0]
    dst[n - 1] = dst[n // 2]
    src[n - 2] = dst[2]
    src[3] = 2 * n + 9
    dst[n - 5] = 2 ** 31 - 1
    src[9], dst[11] = -1, -(2 ** 31)
    dst[n - 9] = src[n - 9]
    c.copy_pages(ints(src), ints(dst))
    m.copy_pages(src, dst)
    m.check(c)
    with pytest.raises(ValueError, match="pair"):
        c.check_status()
    c.check_status()


def test_more_pairs_than_the_pool_has_pages():
    c = make(pages=300, heads=1, layers=2)
    m = ModelCache(c)
    rng = random.Random(1)
    src = [rng.randrange(0, 150) for _ in range(4000)]
    dst = [-1] * 4000
    for at, d in zip(rng.sample(range(4000), 100), range(150, 250)):
        dst[at] = d
    dst[5] = dst[3990] = 299
    c.copy_pages(ints(src), ints(dst))
    m.copy_pages(src, dst)
    m.check(c)
    with pytest.raises(ValueError, match="page 299 is also"):
        c.check_status()


def test_a_fork_into_thousands_of_slots():
    """As many children as a list holds, tails among them, into slots whose last extend was refused; and one page too few."""
    c = make(pages=4200, heads=1, layers=1, seqs=4120, width=3)
    new = [16 * (i % 3) + i % 5 for i in range(20)]  # no tail for every fifth, none at all for some
    c.extend(ints(list(range(20))), ints(new))
    m = ModelCache(c)
    rng = random.Random(2)
    children = rng.sample(range(20, 4120), 4096)
    parents = [i % 20 for i in range(4096)]
    c.extend(ints(children[:50]), ints([99] * 50))
    c.fork(ints(parents), ints(children))
    assert m.fork(parents, children)
    m.check(c)
    m.invariants()
    k, v = values(4096, 1, 1, 64, torch.bfloat16, 3)
    c.write(k, v, ints(children), n_new=ints([1 if new[p] % 16 else 0 for p in parents]))
    m.write(k, v, children, [1 if new[p] % 16 else 0 for p in parents], 0)
    m.check(c)
    with pytest.raises(ValueError, match="too few"):
        c.check_status()
    c.free(ints(children))
    m.free(children)
    spare = m.refs.count(0)
    c.extend(ints(children[-40:]), ints([33] * 40))
    assert m.extend(children[-40:], [33] * 40)
    tails = [p for p in range(20) if new[p] % 16]
    parents = [tails[i % len(tails)] for i in range(spare - 120 + 1)]
    c.fork(ints(parents), ints(children[:len(parents)]))
    assert not m.fork(parents, children[:len(parents)])
    m.check(c)
    with pytest.raises(RuntimeError, match=f"{len(parents)} pages were asked for, {len(parents) - 1} are free"):
        c.check_status()


@pytest.mark.parametrize("page", [16, 128])
def test_rows_that_are_full_to_the_last_entry(page):
    c = make(pages=30, page=page, seqs=5, width=4)
    m = ModelCache(c)
    k, v = values(2, 2, 4 * page, 64, torch.bfloat16, 4)
    c.extend(ints([4, 1]), ints([4 * page, 4 * page - 1]))
    assert m.extend([4, 1], [4 * page, 4 * page - 1])
    c.write(k, v, ints([4, 1]), n_new=ints([4 * page, 4 * page - 1]))
    m.write(k, v, [4, 1], [4 * page, 4 * page - 1], 0)
    c.fork(ints([4, 1]), ints([0, 2]))
    assert m.fork([4, 1], [0, 2])
    c.extend(ints([2, 4]), ints([1, 0]))
    assert m.extend([2, 4], [1, 0])
    c.compact()
    m.compact()
    m.check(c)
    m.invariants()
    c.check_status()
