"""CPU: pages shared between slots (allocator bookkeeping), the grouping of a batch by shared prefixes, and the host
checks of the entry points for shared-prefix attention, step tables and sampling."""

import ctypes
import random

import pytest
import torch

from fpkv import _lib
from fpkv.attention import CausalDecodeMask, PrefixGroups
from fpkv.engine_glue import decoding_block_mask
from fpkv.paged_attention import PagedKVCache
from fpkv.sampling import _per_row, sample


def cpu_cache(n_pages=64, page_size=16, slots=12):
    return PagedKVCache(n_pages, page_size, slots, 2, 64, 1, torch.float32, "cpu")


def check_tables(c, held):
    """Host lists and (CPU) device tables against the model: `held` maps slot -> pages."""
    used = {pg for pages in held.values() for pg in pages}
    assert sorted(c.free_pages) == sorted(set(range(1, c.n_pages)) - used)
    assert len(set(c.free_pages)) == len(c.free_pages)
    for s in range(1, c.max_batch_size):
        pages = held.get(s, [])
        assert c.page_table_cpu[s] == pages
        assert c.page_table[s, :len(pages)].tolist() == pages and (c.page_table[s, len(pages):] == -1).all()
        inverse = {int(p): int(c.physical_to_logical[s, p]) for p in (c.physical_to_logical[s] >= 0).nonzero()}
        assert inverse == {p: i for i, p in enumerate(pages)}


def test_shared_pages_return_with_their_last_holder():
    c = cpu_cache()
    a = c.allocate(); c.reserve(a, None, 5 * 16)
    pa = list(c.page_table_cpu[a])
    b = c.share_prefix(a, 3 * 16); c.reserve(b, None, 4 * 16 + 1)
    assert c.page_table_cpu[b][:3] == pa[:3] and not set(c.page_table_cpu[b][3:]) & set(pa) and c.capacity[b] == 5 * 16
    pb = list(c.page_table_cpu[b])
    d = c.share_prefix(b, 4 * 16)                       # a chain: three of a's pages, one of b's
    held = {a: pa, b: pb, d: pb[:4]}
    check_tables(c, held)
    c.erase(a); del held[a]; check_tables(c, held)
    c.erase(b); del held[b]; check_tables(c, held)
    c.erase(d); del held[d]; check_tables(c, held)
    assert c.num_free_pages == c.n_pages - 1 and not c._page_holders


@pytest.mark.parametrize("seed", range(4))
def test_random_shares_and_erases(seed):
    rng, c, held = random.Random(seed), cpu_cache(), {}
    for _ in range(300):
        what = rng.choice(["new", "share", "grow", "erase"])
        if what == "new" and c.free_batch_idx:
            held[c.allocate()] = []
        elif what == "share" and held and c.free_batch_idx:
            src = rng.choice(list(held)); n = rng.randint(0, len(held[src]))
            held[c.share_prefix(src, n * 16)] = held[src][:n]
        elif what == "grow" and held:
            s = rng.choice(list(held)); want = (len(held[s]) + rng.randint(0, 4)) * 16
            if c.can_reserve(want, s):
                c.reserve(s, None, want); held[s] = list(c.page_table_cpu[s])
        elif what == "erase" and held:
            s = rng.choice(list(held)); c.erase(s); del held[s]
        check_tables(c, held)
    for s in list(held):
        c.erase(s)
    check_tables(c, {})


def test_share_prefix_refusals():
    c = cpu_cache()
    a = c.allocate(); c.reserve(a, None, 40)
    free = list(c.free_batch_idx)
    for slot, n in ((a, 17), (a, 4 * 16), (0, 16), (a + 1, 0), (c.max_batch_size, 0), (a, -16)):
        with pytest.raises(AssertionError):
            c.share_prefix(slot, n)
    assert c.free_batch_idx == free                     # nothing was taken


def groups_of(c, slots, **kw):
    g = c.prefix_groups(slots, **kw)
    return g.groups.tolist(), g.row_group.tolist()


def test_prefix_groups():
    c = cpu_cache(n_pages=200, slots=40)
    doc = c.allocate(); c.reserve(doc, None, 8 * 16)
    pic = c.allocate(); c.reserve(pic, None, 2 * 16)
    asks = [c.share_prefix(doc, 8 * 16) for _ in range(3)]
    for s in asks:
        c.reserve(s, None, 8 * 16 + 5)
    looks = [c.share_prefix(pic, 16) for _ in range(2)]
    lone = c.allocate(); c.reserve(lone, None, 50)
    assert groups_of(c, asks + looks + [lone], rows=8) == ([[0, 3, 8, 0], [3, 2, 1, 0]], [0, 0, 0, 1, 1, -1, -1, -1])
    assert groups_of(c, [asks[0], lone, asks[1]]) == ([], [-1, -1, -1])          # not next to each other
    assert groups_of(c, []) == ([], [])
    # a row that shares one page only does not cut a long common prefix down to that page
    short = c.share_prefix(doc, 16)
    assert groups_of(c, asks + [short])[0] == [[0, 3, 8, 0]]
    assert groups_of(c, asks[:1] + [short])[0] == [[0, 2, 1, 0]]
    # refilled in place
    g = c.prefix_groups(asks + looks + [lone], rows=8)
    at = g.groups.data_ptr()
    c.prefix_groups([lone] + asks, rows=8, into=g)
    assert g.groups.data_ptr() == at and g.groups.tolist() == [[1, 3, 8, 0], [0, 0, 0, 0]]
    assert g.row_group.tolist() == [-1, 0, 0, 0, -1, -1, -1, -1]
    with pytest.raises(AssertionError):
        c.prefix_groups(asks, rows=2)
    with pytest.raises(AssertionError):
        c.prefix_groups(asks, into=g)                   # another number of rows


def test_step_mask_carries_the_groups():
    c = cpu_cache()
    bi, ip = torch.tensor([1]), torch.tensor([0])
    g = PrefixGroups(torch.zeros((0, 4), dtype=torch.int32), torch.full((1,), -1, dtype=torch.int32))
    m = decoding_block_mask(CausalDecodeMask(4, 64, 16), bi, ip, g)
    assert c.convert_logical_block_mask(m, bi).shared is g
    assert CausalDecodeMask(4, 64, 16).for_step(bi, ip).shared is None


# ------------------------------------------------------------------- host checks
def _pool(**kw):
    buf = torch.zeros(64, dtype=torch.int64)
    d = dict(data=buf.data_ptr(), page_table=buf.data_ptr(), physical_to_logical=buf.data_ptr(), num_layers=1,
             n_heads=2, n_pages=4, page_size=128, head_dim=64, max_batch_size=3, dtype=_lib.FPKV_BF16, split_q_heads=0)
    d.update(kw)
    return _lib.FpkvPool(**d), buf


def test_shared_attention_validation():
    L = _lib.lib
    p, buf = _pool()
    ptr, need = buf.data_ptr(), ctypes.c_size_t(0)

    def call(pool=p, out=ptr, q=ptr, sb=256, hq=4, B=2, pt=0, groups=ptr, n=1, rg=ptr, ws=ptr, size=1 << 40, scale=0.125):
        return L.fpkv_decode_attn_shared(ctypes.byref(pool), 0, out, ptr, q, sb, 64, ptr, ptr, pt, B, hq, groups, n, rg,
                                         scale, ws, size, None, None, None)
    assert call(_pool(dtype=_lib.FPKV_F32)[0]) == -7
    assert call(_pool(page_size=64)[0]) == -2 and call(_pool(split_q_heads=4)[0]) == -2
    assert call(_pool(head_dim=96)[0]) == -2
    assert call(hq=3) == -2 and call(hq=34) == -2 and call(n=_lib.MAX_GROUPS + 1) == -2
    assert call(B=-1) == -1 and call(n=-1) == -1 and call(pt=2) == -1 and call(hq=0) == -1
    assert call(out=0) == -1 and call(q=0) == -1 and call(groups=0) == -1 and call(rg=0) == -1 and call(ws=0) == -1
    assert call(q=ptr + 2) == -3 and call(sb=100) == -3 and call(groups=ptr + 4) == -3 and call(rg=ptr + 2) == -3
    assert call(ws=ptr + 8) == -3 and call(size=64) == -6
    assert call(scale=0.0) == -1 and call(scale=-1.0) == -1
    assert call(B=0) == 0
    assert L.fpkv_decode_shared_workspace_bytes(ctypes.byref(p), 2, 4, 1, ctypes.byref(need)) == 0 and need.value > 0
    assert L.fpkv_decode_shared_workspace_bytes(ctypes.byref(p), 2, 4, 1, None) == -1
    assert L.fpkv_decode_shared_workspace_bytes(ctypes.byref(p), 2, 3, 1, ctypes.byref(need)) == -2
    if not torch.cuda.is_available():
        assert call() == -4


def test_step_tables_validation():
    L = _lib.lib
    p, buf = _pool()
    ptr = buf.data_ptr()
    out = _lib.FpkvStepOut(*([ptr] * 8))

    def call(slots=ptr, n=2, row=8, align=4, width=2, tokens=ptr, nt=8, o=out):
        return L.fpkv_step_tables(ctypes.byref(p), slots, ptr, ptr, n, row, align, width, tokens, nt, 0,
                                  ctypes.byref(o) if o is not None else None, None, None)
    assert call(n=-1) == -1 and call(row=-1) == -1 and call(align=0) == -1 and call(width=-1) == -1 and call(nt=-1) == -1
    assert call(slots=0) == -1 and call(o=None) == -1 and call(tokens=0) == -1
    assert call(n=_lib.MAX_REQUESTS + 1) == -2 and call(row=(1 << 30) + 1) == -2
    assert call(slots=ptr + 4) == -3 and call(tokens=ptr + 4) == -3
    assert call(o=_lib.FpkvStepOut(ptr + 4)) == -3
    if not torch.cuda.is_available():
        assert call() == -4


def test_sample_validation():
    L = _lib.lib
    buf = torch.zeros(64, dtype=torch.int64)
    ptr = buf.data_ptr()

    def call(x=ptr, dt=_lib.FPKV_BF16, stride=100, rows=2, vocab=100, u=ptr, t=None, k=None, tok=ptr, lp=ptr):
        return L.fpkv_sample(x, dt, stride, rows, vocab, u, t, k, None, None, tok, lp, None)
    assert call(dt=5) == -7 and call(rows=-1) == -1 and call(vocab=0) == -1
    assert call(stride=99) == -2 and call(vocab=(1 << 24) + 1, stride=1 << 25) == -2
    assert call(x=0) == -1 and call(u=0) == -1 and call(tok=0) == -1
    assert call(x=ptr + 1) == -3 and call(dt=_lib.FPKV_F32, x=ptr + 2) == -3 and call(t=ptr + 2) == -3
    assert call(k=ptr + 2) == -3 and call(tok=ptr + 4) == -3 and call(lp=ptr + 2) == -3
    assert call(rows=0) == 0
    if not torch.cuda.is_available():
        assert call() == -4 and call(rows=1, stride=0) == -4


def test_python_refusals():
    x, u = torch.zeros(2, 8), torch.zeros(2)
    for bad in (lambda: sample(x[0], u), lambda: sample(x.long(), u), lambda: sample(x, u[:1]), lambda: sample(x, u.double()),
                lambda: sample(x[:, :0], u)):
        with pytest.raises(AssertionError):
            bad()
    with pytest.raises(RuntimeError, match="CUDA"):
        sample(x, u)
    c = cpu_cache()
    i64, i32 = torch.zeros(2, dtype=torch.int64), torch.zeros(2, dtype=torch.int32)
    for bad in (lambda: c.step_tables(i32, i32, i32, 8), lambda: c.step_tables(i64, i64, i32, 8),
                lambda: c.step_tables(i64, i32, i32[:1], 8), lambda: c.step_tables(i64, i32, i32, -1),
                lambda: c.step_tables(i64, i32, i32, 8, align=0), lambda: c.step_tables(i64, i32, i32, 8, tokens=i32)):
        with pytest.raises(AssertionError):
            bad()
    with pytest.raises(RuntimeError, match="CUDA"):
        c.step_tables(i64, i32, i32, 8)


def test_prefix_groups_beyond_the_room_left_out():
    """A record has room for so many groups; those that save least are in none, in a new record and in a refilled one."""
    n = _lib.MAX_GROUPS + 6
    c = PagedKVCache(4 * n, 16, 3 * n, 1, 64, 1, torch.float32, "cpu")
    slots, first = [], []
    for i in range(n):
        pages = 2 if i % 200 else 1                     # the groups of one page save least: 0, 200, ... 1000
        a = c.allocate(); c.reserve(a, None, pages * 16)
        first.append(len(slots)); slots += [a, c.share_prefix(a, pages * 16)]
    g = c.prefix_groups(slots)
    assert g.n_groups == _lib.MAX_GROUPS
    kept = [i for i in range(n) if i % 200]
    assert g.groups.tolist() == [[first[i], 2, 2, 0] for i in kept]
    assert g.row_group.tolist() == [k for i in range(n) for k in 2 * [kept.index(i) if i % 200 else -1]]
    small = c.prefix_groups(slots[:4], rows=8)           # room for two
    assert small.n_groups == 2
    c.prefix_groups(slots[:8], into=small)
    assert small.groups.tolist() == [[2, 2, 2, 0], [4, 2, 2, 0]] and small.row_group.tolist() == [-1, -1, 0, 0, 1, 1, -1, -1]
    with pytest.raises(AssertionError):
        c.prefix_groups(slots[:2], into=small)           # another number of rows


def test_prefix_groups_refuse_slots_that_are_none():
    c = cpu_cache()
    a = c.allocate(); c.reserve(a, None, 40)
    for bad in ([a, -1], [-1, -1], [a, c.max_batch_size]):
        with pytest.raises(AssertionError):
            c.prefix_groups(bad)
    assert groups_of(c, [a, 0, 0]) == ([], [-1, -1, -1])         # padding is fine


def test_top_k_as_a_number_of_any_size():
    like = torch.zeros(3, 1000)
    for k, want in ((2 ** 40, 1000), (2 ** 31, 1000), (1000, 1000), (7, 7), (0, 0), (-1, 0), (-2 ** 40, 0)):
        got = _per_row(k, "top_k", 3, torch.int32, like)
        assert got.dtype == torch.int32 and got.tolist() == [want] * 3
        assert torch.equal(got, _per_row(torch.full((3,), k), "top_k", 3, torch.int32, like))


def test_launches_go_to_the_caches_device(monkeypatch):
    """With another device current, queued table edits and calls with groups, those that are served row by row among them, switch
    to the cache's (stand-ins for CUDA: the device current at the launch is what counts)."""
    current, seen = [0], []

    class Device:
        def __init__(self, d):
            self.d = d if isinstance(d, int) else d.index

        def __enter__(self):
            self.was, current[0] = current[0], self.d

        def __exit__(self, *a):
            current[0] = self.was

    class Event:
        def record(self, stream):
            pass

        def synchronize(self):
            pass

    class Stop(Exception):
        pass

    class Query:
        is_cuda = True

        def get_device(self):
            return 1

        @property
        def shape(self):
            seen.append(current[0])
            raise Stop

    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: None)
    monkeypatch.setattr("fpkv.paged_attention._stream", lambda d: 0)

    class Library:
        @staticmethod
        def fpkv_alloc_step(*a):
            seen.append(current[0])
            return 0

    c = cpu_cache()
    c._dev = torch.device("cuda", 1)
    c._ops_cap, c._ops_turn, c._alloc = 8, 0, _lib.FpkvAllocState()
    c._ops_host, c._ops_done, c._ops_dev = [torch.empty(8, 4, dtype=torch.int32)] * 2, [Event(), Event()], torch.empty(8, 4, dtype=torch.int32)
    a = c.allocate(); c.reserve(a, None, 40); c.share_prefix(a, 32)
    monkeypatch.setattr(_lib, "lib", Library)
    c.flush_tables()
    assert seen == [1] and current == [0] and not c._pending
    g = PrefixGroups(torch.zeros((0, 4), dtype=torch.int32), torch.full((1,), -1, dtype=torch.int32))
    for call in (lambda: c.decode_attention(0, Query(), None, None, shared=g), lambda: c.decode_step(0, Query(), None, None, None, None, shared=g)):
        with pytest.raises(Stop):
            call()
    assert seen == [1, 1, 1] and current == [0]
