"""Refusals of the paged cache that need no device: the C entry points check before they launch, the Python side before it calls."""

import ctypes as C

import pytest
import torch

from fa4b import PagedKVCache, _lib


def good(**change):
    f = dict(k=0x10000, v=0x20000, k_layer_stride=100 * 8 * 16 * 128, k_page_stride=8 * 16 * 128, v_layer_stride=100 * 8 * 16 * 128,
             v_page_stride=8 * 16 * 128, layers=2, num_pages=100, Hkv=8, page_tokens=16, D=128, dtype=0, k_scale=0, v_scale=0, page_table=0x30000,
             table_stride=50, max_seqs=10, table_width=50, seq_lens=0x40000, ref_counts=0x50000, work=0x60000)
    return _lib.KvCache(**(f | change))


@pytest.mark.parametrize("change,status,text", [
    (dict(D=96), 1, b"head dim"), (dict(page_tokens=24), 1, b"pages of 24"), (dict(page_tokens=0), 1, b"pages of 0"), (dict(dtype=3), 3, b"dtype"),
    (dict(dtype=2), 6, b"k_scale"), (dict(k=0), 6, b"NULL"), (dict(k=0x10008), 2, b"16-byte"), (dict(work=0x60004), 2, b"16-byte"), (dict(work=0), 6, b"NULL"),
    (dict(max_seqs=1 << 20), 1, b"max_seqs"), (dict(table_width=1 << 19, table_stride=1 << 19), 1, b"table_width"), (dict(layers=0), 1, b"positive"),
    (dict(num_pages=-1), 1, b"positive"), (dict(table_stride=49), 1, b"overlap"), (dict(k_page_stride=8), 1, b"overlap"), (dict(v_layer_stride=12), 2, b"multiples"),
])
def test_every_call_refuses_a_bad_cache(change, status, text):
    h = _lib.lib()
    c = good(**change)
    w = _lib.KvWriteArgs(0x1000, 0x1000, _lib.Strides(), _lib.Strides(), 1, 0, 0, 1, 0x1000, 0)
    for got in (h.fa4b_kv_free(C.addressof(c), 0x1000, 1, 0), h.fa4b_kv_extend(C.addressof(c), 0x1000, 0x1000, 1, 0),
                h.fa4b_kv_fork(C.addressof(c), 0x1000, 0x1000, 1, 0), h.fa4b_kv_copy_pages(C.addressof(c), 0x1000, 0x1000, 1, 0),
                h.fa4b_kv_compact(C.addressof(c), 0), h.fa4b_kv_write(C.addressof(c), C.addressof(w), 0), h.fa4b_kv_check_status(C.addressof(c), 0)):
        assert got == status and text in h.fa4b_last_error()


@pytest.mark.parametrize("which", ["k_layer_stride", "v_layer_stride"])
def test_layers_that_lie_on_one_another_are_refused(which):
    h = _lib.lib()
    block = 8 * 16 * 128
    for stride, status in ((0, 1), (block - 128, 1), (block, 0)):
        c = good(**{which: stride})
        assert h.fa4b_kv_free(C.addressof(c), 0, 0, 0) == status and (status == 0 or b"layers overlap" in h.fa4b_last_error())
    c = good(layers=1, **{which: 0})  # one layer: the stride says nothing
    assert h.fa4b_kv_free(C.addressof(c), 0, 0, 0) == 0


def test_rows_of_the_result_that_lie_on_one_another_are_refused():
    h = _lib.lib()
    c, z = good(), _lib.Strides(1024, 128, 128)

    def call(o_strides, n=2, T=2):
        a = _lib.AttnPagedArgs(q=0x1000, q_strides=z, o=0x2000, o_strides=o_strides, lse=0x3000, n=n, T=T, Hq=8, layer=0, q_dtype=0, softmax_scale=0.0, seqs=0x4000,
                               groups=0, group_offsets=0, shared_lens=0, ws=0x10000)
        return h.fa4b_attn_paged_workspace_bytes(C.addressof(c), C.addressof(a))

    for bad in ((0, 128, 1024), (2048, 0, 1024), (2048, 128, 0)):
        assert call(_lib.Strides(*bad)) == 0 and b"one another" in h.fa4b_last_error()
    assert call(_lib.Strides(2048, 128, 1024)) > 0 and call(_lib.Strides(0, 128, 0), n=1, T=1) > 0


def test_lists_and_arguments_are_checked():
    h = _lib.lib()
    c = good()
    at = C.addressof(c)
    assert h.fa4b_kv_free(None, 0x1000, 1, 0) == 6
    assert h.fa4b_kv_free(at, 0x1000, -1, 0) == 1 and h.fa4b_kv_free(at, 0x1000, 4097, 0) == 1 and b"4096" in h.fa4b_last_error()
    assert h.fa4b_kv_free(at, 0, 1, 0) == 6 and h.fa4b_kv_extend(at, 0x1000, 0, 1, 0) == 6 and h.fa4b_kv_fork(at, 0, 0x1000, 1, 0) == 6
    assert h.fa4b_kv_free(at, 0, 0, 0) == 0 and h.fa4b_kv_copy_pages(at, 0, 0, 0, 0) == 0  # nothing to do
    s = _lib.Strides(8, 8, 8)

    def write(**change):
        f = dict(k_new=0x1000, v_new=0x1000, k_strides=s, v_strides=s, T=1, src_dtype=0, layer=0, n=1, seqs=0x1000, n_new=0)
        w = _lib.KvWriteArgs(**(f | change))
        return h.fa4b_kv_write(at, C.addressof(w), 0)

    assert write(layer=2) == 1 and write(layer=-1) == 1 and write(T=-1) == 1 and write(T=2 ** 31 - 1) == 1
    assert write(src_dtype=1) == 3 and write(src_dtype=2) == 3
    assert write(k_new=0) == 6 and write(seqs=0) == 6 and write(v_new=0x1008) == 2 and write(k_strides=_lib.Strides(4, 8, 8)) == 2
    assert write(T=0) == 0 and write(n=0) == 0


def test_workspace_bytes_cover_the_lists_of_a_compaction():
    h = _lib.lib()
    for pages in (1, 100, 4096, 4097, 1 << 20):
        c = good(num_pages=pages)
        assert h.fa4b_kv_workspace_bytes(C.addressof(c)) == 4 * (16 + 2 * 4096 + -(-pages // 4096) + 3 * pages)
    assert h.fa4b_kv_workspace_bytes(None) == 0


def test_constants_agree_between_the_header_and_the_python_side():
    import pathlib
    import re

    from fa4b import kv_cache

    header = (pathlib.Path(__file__).resolve().parents[1] / "include" / "fa4b.h").read_text()
    got = {m.group(1): int(m.group(2)) for m in re.finditer(r"(FA4B_KV_(?:BF16|F16|E4M3)) = (\d+)", header)}
    assert got == {"FA4B_KV_BF16": 0, "FA4B_KV_F16": 1, "FA4B_KV_E4M3": 2}
    assert kv_cache.KV_DTYPES == {torch.bfloat16: 0, torch.float16: 1, torch.float8_e4m3fn: 2}


def test_the_python_side_refuses_cpu_tensors_and_wrong_types():
    k = torch.zeros(1, 4, 2, 16, 64, dtype=torch.bfloat16)
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        PagedKVCache(k, k.clone(), i[None], i[:1], i)
    with pytest.raises(TypeError, match="float32"):
        PagedKVCache(k.float(), k.float(), i[None], i[:1], i)
    with pytest.raises(ValueError, match="layers"):
        PagedKVCache(k[0], k[0], i[None], i[:1], i)
    with pytest.raises(TypeError, match="dtype"):
        PagedKVCache.empty(4, 16, 2, 64, 3, 3, dtype=torch.float32, device="cpu")
    with pytest.raises(ValueError, match="positive"):
        PagedKVCache.empty(4, 16, 2, 64, 0, 3, device="cpu")


def test_attention_over_the_cache_is_refused_before_a_launch():
    h = _lib.lib()
    z = _lib.Strides(1024, 128, 128)

    def call(cache=None, **change):
        f = dict(q=0x1000, q_strides=z, o=0x2000, o_strides=z, lse=0x3000, n=2, T=1, Hq=32, layer=0, q_dtype=0, softmax_scale=0.0, seqs=0x4000, groups=0,
                 group_offsets=0, shared_lens=0, ws=0x10000)
        a = _lib.AttnPagedArgs(**(f | change))
        c = cache or good()
        return h.fa4b_attn_paged_fwd(C.addressof(c), C.addressof(a), 0), h.fa4b_attn_paged_workspace_bytes(C.addressof(c), C.addressof(a)), h.fa4b_last_error()

    for change, status, text in ((dict(n=-1), 1, b"n=-1"), (dict(n=5000), 1, b"n=5000"), (dict(T=0), 1, b"T=0"), (dict(T=17), 1, b"T=17"),
                                 (dict(Hq=12), 1, b"multiple"), (dict(Hq=8 * 129), 1, b"at most 128"), (dict(layer=2), 1, b"layer 2"), (dict(q_dtype=1), 3, b"own type"),
                                 (dict(q_dtype=2), 3, b"bf16 or f16"), (dict(groups=3), 1, b"groups=3"), (dict(groups=1), 6, b"group_offsets"),
                                 (dict(seqs=0, n=11), 1, b"list of slots"), (dict(q=0x1008), 2, b"16-byte"), (dict(o_strides=_lib.Strides(4, 8, 8)), 2, b"multiples of 8")):
        got, size, error = call(**change)
        assert got == status and size == 0 and text in error, change
    for scale in (float("nan"), float("inf"), float("-inf")):
        got, size, error = call(softmax_scale=scale)
        assert got == 6 and size == 0 and b"finite" in error
    assert call(ws=0)[0] == 6 and call(lse=0)[0] == 6 and call(ws=0x10010)[0] == 2 and call(n=0, q=0, o=0, lse=0, ws=0)[0] == 0
    got, size, error = call(cache=good(table_width=1 << 18, table_stride=1 << 18, page_tokens=128, k_page_stride=1 << 17, v_page_stride=1 << 17, max_seqs=5000), n=4096)
    assert got == 1 and size == 0 and b"too many" in error
    assert call(cache=good(D=96))[0] == 1


def test_packed_arguments_have_the_layout_of_the_structs():
    from fa4b import kv_cache

    for packed, struct in ((kv_cache._WRITE, _lib.KvWriteArgs), (kv_cache._ATTEND, _lib.AttnPagedArgs)):
        assert packed.size == C.sizeof(struct)
        count = len(packed.unpack(bytes(packed.size)))
        values = tuple(float(i) if i == 14 and struct is _lib.AttnPagedArgs else i + 1 for i in range(count))
        got = struct.from_buffer_copy(packed.pack(*values))
        flat = []
        for name, kind in struct._fields_:
            x = getattr(got, name)
            flat += [x.batch, x.head, x.seq] if kind is _lib.Strides else [x]
        assert tuple(flat) == values


def _kernels(name):
    """Every kernel of a source file: name, parameters, body."""
    import pathlib
    import re

    text = (pathlib.Path(_lib.__file__).resolve().parents[1] / "csrc" / name).read_text()
    text = re.sub(r"//[^\n]*", "", text)
    for m in re.finditer(r"__global__ void (?:__launch_bounds__\([^\n]*?\) )?(\w+)\(([^{]*?)\) \{\n(.*?)\n\}\n", text, re.S):
        yield m.groups()


def test_kernels_that_come_up_early_wait_before_they_read():
    """A launch that overlaps the one before sees what earlier launches wrote behind its own wait only, also what an even earlier one has
    long written: nothing but the arguments is looked at before it."""
    import re

    memory = re.compile(r"\bp\.(seq|head|group|seqs|offsets|shared|q|k_scale|own_acc|own_ml|own_cum|g_cum|prefix_acc|prefix_ml)\b|\bc\.(lens|table|refs|work(?! \+)|k|v)\b|"
                        r"\b(seqs|n_new|parents|children|src|dst)\[|paged_small|\.start\(|tma_load")
    seen = set()
    for name in ("kv_cache.cu", "attn_paged.cu", "attn_prefix.cu"):
        for kernel, _, body in _kernels(name):
            before, wait, _ = body.partition("pdl_wait();")
            assert wait, kernel
            assert not memory.search(before), (kernel, memory.search(before))
            seen.add(kernel)
    assert {"paged_plan_kernel", "attn_prefix_kernel", "attn_solo_kernel", "attn_team_kernel", "paged_join_kernel", "kv_extend_kernel", "kv_copy_kernel"} <= seen and len(seen) == 15, seen


def test_kernels_that_come_up_early_promise_nothing_about_their_lists():
    """`const T* __restrict__` tells the compiler that nobody writes the list while the kernel runs, so that its loads may move above the wait;
    the kernel that writes it may still be running then."""
    for name in ("kv_cache.cu", "attn_paged.cu", "attn_prefix.cu"):
        for kernel, parameters, _ in _kernels(name):
            assert "__restrict__" not in parameters, kernel


def test_unknown_flags_of_the_attention_are_refused():
    h = _lib.lib()
    z = _lib.Strides(1024, 128, 128)
    c = good()
    for flags, ok in ((0, True), (1, True), (2, True), (3, True), (4, False), (-1, False)):
        a = _lib.AttnPagedArgs(q=0x1000, q_strides=z, o=0x2000, o_strides=z, lse=0x3000, n=2, T=1, Hq=8, layer=0, q_dtype=0, softmax_scale=0.0, seqs=0x4000, groups=0,
                               flags=flags, group_offsets=0, shared_lens=0, ws=0x10000)
        assert (h.fa4b_attn_paged_workspace_bytes(C.addressof(c), C.addressof(a)) > 0) == ok
        assert ok or b"flags" in h.fa4b_last_error()
    assert C.sizeof(_lib.AttnPagedArgs) == 136 and _lib.AttnPagedArgs.group_offsets.offset == 112  # what stands around the flags is where it was


def _pages_overlap(layer, page, layers, pages, block):
    at = sorted(i * layer + j * page for i in range(layers) for j in range(pages))
    return any(b - a < block for a, b in zip(at, at[1:]))


def test_pools_whose_layers_share_pages_are_refused_by_every_call_that_writes_them():
    """Every layout of a few layers and pages against the list of their places; K and V on their own."""
    h = _lib.lib()
    block = 2 * 16 * 64
    w = _lib.KvWriteArgs(0x1000, 0x1000, _lib.Strides(), _lib.Strides(), 0, 0, 0, 1, 0x1000, 0)
    seen = set()
    for layers, pages in ((2, 100), (3, 2), (4, 5), (2, 2), (1, 9), (7, 1)):
        for layer in (block, block + 64, 2 * block, 3 * block, 5 * block, 5 * block + 64, (pages - 1) * block + block, 100 * block, 3 * pages * block):
            for page in (block, block + 8, 2 * block, 3 * block + 64, layers * block, (layers - 1) * layer + block):
                bad = _pages_overlap(layer, page, layers, pages, block)
                for which in "kv":
                    c = good(Hkv=2, D=64, layers=layers, num_pages=pages, **{f"{x}_{y}_stride": z for x in "kv" for y, z in (("layer", 1000 * block), ("page", block))}
                             | {f"{which}_layer_stride": layer, f"{which}_page_stride": page})
                    at = C.addressof(c)
                    for got in (h.fa4b_kv_copy_pages(at, 0, 0, 0, 0), h.fa4b_kv_fork(at, 0, 0, 0, 0), h.fa4b_kv_write(at, C.addressof(w), 0)):
                        assert got == bad and (not bad or b"layers overlap" in h.fa4b_last_error()), (layers, pages, layer, page)
                    if bad:
                        assert h.fa4b_kv_compact(at, 0) == 1
                seen.add(bad)
    assert seen == {False, True}


def test_the_workspace_is_sized_for_the_device_of_the_cache(monkeypatch):
    """Pieces of work, and with them the workspace, are as many as the device has room for: the cache's, not the current one."""
    import contextlib
    import types

    from fa4b import kv_cache

    current, asked = [1], []

    @contextlib.contextmanager
    def device(index):
        before, current[0] = current[0], index
        yield
        current[0] = before

    def answer(*_):
        asked.append(current[0])
        return 1024

    c = PagedKVCache.__new__(PagedKVCache)
    c.device, c._index, c._d, c._takes, c._ws_bytes, c._at = torch.device("cpu"), -1, 64, (torch.bfloat16,), {}, 0
    c._floats = torch.zeros(0)
    c._lib = types.SimpleNamespace(fa4b_attn_paged_workspace_bytes=answer, fa4b_attn_paged_fwd=lambda *_: asked.append(current[0]) or 0)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(kv_cache, "_current_device", lambda: current[0])
    monkeypatch.setattr(kv_cache, "_raw_stream", lambda index: 0)
    for _ in range(2):
        c.attend(torch.zeros(2, 4, 1, 64, dtype=torch.bfloat16))
    assert asked == [-1, -1, -1] and current == [1]
