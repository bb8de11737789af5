"""GPU: decode attention of a batch that shares prefixes, against a 64-bit computation over every row's own keys."""

import ctypes
import math

import pytest
import torch

from fpkv import _lib
from fpkv.paged_attention import PagedKVCache, paged_attention

pytestmark = pytest.mark.gpu
P = 128


def build(Hq, Hkv, D, dtype, groups, spare=(), seed=0, layers=1, layer=0, max_pages=None, page_size=P):
    """groups: list of (shared pages, [tokens of each row]); a row's tokens count from its first key, so they may end
    inside the prefix.  spare: tokens of rows that share nothing.  Everything that no sequence appended -- the tails of
    last pages, free pages -- is NaN.  Returns the cache, slots and last positions."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    need = 1 + sum(n + sum(max(0, -(-t // page_size) - n) for t in rows) for n, rows in groups) + sum(-(-t // page_size) for t in spare)
    n_pages = max_pages or need + 3
    B = sum(len(r) for _, r in groups) + len(spare)
    c = PagedKVCache(n_pages, page_size, B + 1, Hkv, D, layers, dtype, "cuda")
    c.free_pages = (torch.randperm(n_pages - 1, generator=torch.Generator().manual_seed(seed)) + 1).tolist()
    slots, last = [], []
    for n, rows in groups:
        first = None
        for t in rows:
            if first is None:
                s = first = c.allocate(); c.reserve(s, None, n * page_size)
            else:
                s = c.share_prefix(first, n * page_size)
            c.reserve(s, None, t)
            slots.append(s); last.append(t - 1)
    for t in spare:
        s = c.allocate(); c.reserve(s, None, t); slots.append(s); last.append(t - 1)
    c.kv_cache.fill_(float("nan"))
    written = {}
    for s, p in zip(slots, last):                        # the pages of a prefix are filled by whoever reads furthest
        for j, pg in enumerate(c.page_table_cpu[s]):
            written[pg] = max(written.get(pg, 0), min(page_size, p + 1 - j * page_size))
    at = 0
    for n, rows in groups:                               # ... and wholly, being a prefix
        for pg in c.page_table_cpu[slots[at]][:n]:
            written[pg] = page_size
        at += len(rows)
    pool = c.kv_cache[layer, :, 0]
    for pg, n in written.items():
        if n > 0:
            pool[:, :, pg * page_size:pg * page_size + n] = torch.randn(2, Hkv, n, D, generator=gen, device="cuda").to(dtype)
    q = torch.randn(B, Hq, 1, D, generator=gen, device="cuda").to(dtype)
    return c, slots, last, q


def reference(c, layer, q, slots, last, scale=None):
    """64-bit attention of every row over its own pages, and bounds of the kernel's error.  Scores: products of 16-bit
    numbers summed in 32 bits (at most D half-steps of the sum of magnitudes, and as many for the scaling); weights: that,
    a 32-bit exponential (2^-21) and one rounding to 16 bits; output: one rounding."""
    B, Hq, _, D = q.shape
    H, eps = c.n_heads, torch.finfo(q.dtype).eps / 2
    scale = 1 / math.sqrt(D) if scale is None else scale
    out, lse = torch.zeros(B, Hq, 1, D, dtype=torch.double), torch.full((B, Hq, 1), -math.inf, dtype=torch.double)
    tol_o, tol_l = torch.zeros_like(out), torch.zeros_like(lse)
    for b, (s, p) in enumerate(zip(slots, last)):
        pages = torch.tensor(c.page_table_cpu[s], device="cuda")
        if s == 0 or p < 0 or not len(pages):
            continue
        rows = (pages[:, None] * c.page_size + torch.arange(c.page_size, device="cuda")).reshape(-1)[:p + 1]
        k, v = c.kv_cache[layer, 0, 0][:, rows].double(), c.kv_cache[layer, 1, 0][:, rows].double()
        qb = q[b, :, 0].double().view(H, Hq // H, D)
        x = torch.einsum("hrd,hkd->hrk", qb, k) * scale
        off = (D + 8) * 2.0 ** -24 * (torch.einsum("hrd,hkd->hrk", qb.abs(), k.abs()) * abs(scale)).amax(-1, keepdim=True) + 2.0 ** -21
        l = torch.logsumexp(x, -1, keepdim=True)
        w = torch.exp(x - l)
        o = torch.einsum("hrk,hkd->hrd", w, v)
        mean = torch.einsum("hrk,hkd->hrd", w, v.abs())
        out[b, :, 0] = o.reshape(Hq, D).cpu(); lse[b] = l.reshape(Hq, 1).cpu()
        tol_o[b, :, 0] = ((eps + 4 * off) * mean + eps * o.abs()).reshape(Hq, D).cpu() + 1e-7
        tol_l[b] = (off + 2.0 ** -22 * (1 + l.abs())).reshape(Hq, 1).cpu()
    return out, lse, tol_o, tol_l


def check(out, lse, ref, what=""):
    r_out, r_lse, tol_o, tol_l = ref
    out, lse = out.double().cpu(), lse.double().cpu()
    assert out.shape == r_out.shape and lse.shape == r_lse.shape
    dead = r_lse == -math.inf
    assert torch.equal(lse == -math.inf, dead), what
    assert (out[dead.expand(out.shape[:-1])] == 0).all(), what
    assert not out.isnan().any(), f"{what}: NaN"
    excess = ((out - r_out).abs() / tol_o.clamp(min=1e-12)).max().item()
    assert excess <= 1, f"{what}: output is {excess:.2f} times its bound off"
    d = torch.where(dead, torch.zeros_like(lse), (lse - r_lse).abs() / tol_l.clamp(min=1e-12)).max().item()
    assert d <= 1, f"{what}: lse is {d:.2f} times its bound off"


def run(c, slots, last, q, layer=0, rows=None, pos_dtype=torch.int32, **kw):
    bi = torch.tensor(slots, device="cuda")
    ip = torch.tensor(last, dtype=pos_dtype, device="cuda")
    g = c.prefix_groups(slots)
    out, lse = c.decode_attention(layer, q, bi, ip, shared=g, **kw)
    torch.cuda.synchronize()
    c.check_status()
    return out, lse, g


SHAPES = [(16, 8, 128, torch.bfloat16), (4, 2, 64, torch.float16), (4, 4, 128, torch.bfloat16), (8, 1, 64, torch.bfloat16),
          (6, 2, 128, torch.float16), (16, 1, 128, torch.bfloat16), (5, 1, 64, torch.float16), (8, 2, 128, torch.float16)]
BATCHES = {
    "two rows, one page": ([(1, [129, 130])], ()),
    "own part empty": ([(2, [256, 256, 300])], ()),
    "positions inside the prefix": ([(4, [700, 1, 128, 129, 511, 512, 513])], ()),
    "odd sizes and spare rows": ([(3, [385, 400, 777]), (1, [200, 128]), (7, [900] * 5)], (1, 128, 129, 1500)),
    "wide group": ([(2, [257 + i for i in range(70)])], (40,)),
    "very wide group": ([(1, [129 + (i % 5) for i in range(150)]), (3, [390] * 3)], ()),
    "odd shares": ([(53, [53 * 128 + 5 * i + 1 for i in range(3)]), (5, [700, 701]), (1, [140, 300])], (77,)),
    "long prefix": ([(65, [65 * 128 + 1 + 50 * i for i in range(4)])], (9000,)),
}


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}x{s[1]}x{s[2]}-{str(s[3])[6:]}")
@pytest.mark.parametrize("batch", BATCHES, ids=lambda b: b.replace(" ", "-"))
def test_against_64_bits(shape, batch):
    c, slots, last, q = build(*shape, *BATCHES[batch], seed=len(batch))
    out, lse, g = run(c, slots, last, q)
    assert g.n_groups == len(BATCHES[batch][0])
    check(out, lse, reference(c, 0, q, slots, last), batch)


@pytest.mark.parametrize("batch", [([(1, [129 + i % 40 for i in range(600)]), (1, [128 + i % 300 for i in range(480)])], (1, 300)),
                                   ([(1 + g % 3, [500, 400 + g]) for g in range(70)], ())], ids=["more rows than a launch", "many groups"])
def test_large_batches(batch):
    c, slots, last, q = build(4, 2, 64, torch.bfloat16, *batch)
    out, lse, g = run(c, slots, last, q)
    assert g.n_groups == len(batch[0])
    check(out, lse, reference(c, 0, q, slots, last))


def test_agrees_with_the_unshared_path_and_the_call_site():
    c, slots, last, q = build(16, 8, 128, torch.bfloat16, *BATCHES["odd sizes and spare rows"], layers=3, layer=2)
    bi, ip = torch.tensor(slots, device="cuda"), torch.tensor(last, device="cuda")
    plain, plain_lse = c.decode_attention(2, q, bi, ip)
    mask = c.convert_logical_block_mask(c.create_causal_blockmask(len(slots), 2048).for_step(bi, ip, c.prefix_groups(slots)), bi)
    out, lse = paged_attention(q, c, 2, bi, ip, mask)
    c.check_status()
    ref = reference(c, 2, q, slots, last)
    check(out, lse, ref); check(plain, plain_lse, ref)


def test_padding_rows_strides_and_out():
    c, slots, last, q = build(16, 8, 128, torch.bfloat16, [(2, [300, 301, 302])], (70,))
    B, pad = 4, 2
    wide = torch.zeros(B + pad, 2, 16, 1, 128, dtype=q.dtype, device="cuda")
    wide[:B, 1] = q
    qv = wide[:, 1]                                      # rows two heads' blocks apart
    g = c.prefix_groups(slots, rows=B + pad)
    bi = torch.tensor(slots + [0] * pad, dtype=torch.int32, device="cuda")         # converted on the way in
    ip = torch.tensor([[p] for p in last + [0] * pad], device="cuda")
    out = torch.full((B + pad, 16, 1, 128), 7.0, dtype=q.dtype, device="cuda")
    lse = torch.full((B + pad, 16, 1), 7.0, device="cuda")
    got = c.decode_attention(0, qv, bi, ip, out=out, lse=lse, shared=g)
    assert got[0] is out and got[1] is lse
    c.check_status()
    check(out, lse, reference(c, 0, qv, slots + [0] * pad, last + [0] * pad))


def test_one_row_groups_and_groups_without_rows():
    c, slots, last, q = build(4, 2, 128, torch.float16, [(3, [400, 500])], (260,))
    bi, ip = torch.tensor(slots, device="cuda"), torch.tensor(last, dtype=torch.int32, device="cuda")
    g = c.prefix_groups(slots)
    ref = reference(c, 0, q, slots, last)
    for groups, rows in (([[0, 1, 3, 0], [1, 1, 3, 0], [2, 1, 2, 0]], [0, 1, 2]), ([[0, 0, 0, 0], [0, 2, 3, 0], [2, 1, 0, 0]], [1, 1, 2]),
                         ([[0, 2, 3, 0]], [0, 0, -1]), ([[0, 2, 1, 0]], [0, -1, 5]), ([[0, 2, 3, 0], [2, 9, 1, 0]], [0, 0, 1])):
        g.groups = torch.tensor(groups, dtype=torch.int32, device="cuda")
        g.row_group = torch.tensor(rows, dtype=torch.int32, device="cuda")
        out, lse = c.decode_attention(0, q, bi, ip, shared=g)
        c.check_status()
        check(out, lse, ref, str(groups))


def test_one_slot_in_several_rows():
    """The same slot at several positions: all its pages are shared, its last one partly filled, rows end inside it."""
    c, slots, last, q = build(16, 8, 128, torch.bfloat16, [], (700, 130))
    s, p = [slots[0]] * 4 + [slots[1]] * 2, [699, 0, 511, 640, 129, 128]
    q = q[[0, 0, 0, 0, 1, 1]] * torch.arange(1, 7, device="cuda", dtype=q.dtype).view(6, 1, 1, 1) / 4
    out, lse, g = run(c, s, p, q)
    assert g.groups.tolist() == [[0, 4, 6, 0], [4, 2, 2, 0]]
    check(out, lse, reference(c, 0, q, s, p))


def test_no_rows():
    c, slots, last, q = build(4, 2, 64, torch.bfloat16, [(1, [130, 140])], ())
    out, lse = c.decode_attention(0, q[:0], torch.zeros(0, dtype=torch.int64, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda"),
                                  shared=c.prefix_groups([]))
    assert out.shape == (0, 4, 1, 64) and lse.shape == (0, 4, 1)


def test_sink_gate_and_scale():
    c, slots, last, q = build(16, 8, 128, torch.bfloat16, [(2, [300, 310])], ())
    bi, ip = torch.tensor(slots, device="cuda"), torch.tensor(last, dtype=torch.int32, device="cuda")
    g = c.prefix_groups(slots)
    sinks = torch.randn(16, device="cuda")
    out, lse = c.decode_attention(0, q, bi, ip, sm_scale=0.31, shared=g)
    check(out, lse, reference(c, 0, q, slots, last, 0.31))
    gated, lse2 = c.decode_attention(0, q, bi, ip, sm_scale=0.31, sinks=sinks, shared=g)
    want = out.double() * torch.sigmoid(lse.double() - sinks.double()[None, :, None])[..., None]
    # one rounding of the gated value, and the fast exponential of the gate (2^-20)
    assert ((gated.double() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -20) + 1e-30).all()
    assert torch.equal(lse, lse2)


def test_unmapped_pages_and_bad_rows():
    c, slots, last, q = build(4, 2, 128, torch.bfloat16, [(2, [300, 301])], (200, 100))
    bi, ip = torch.tensor(slots, device="cuda"), torch.tensor(last, dtype=torch.int32, device="cuda")
    g = c.prefix_groups(slots)
    # the first row of no group points out of range: it alone is lost
    bad = bi.clone(); bad[3] = 99
    out, lse = c.decode_attention(0, q, bad, ip, shared=g)
    with pytest.raises(RuntimeError, match="bad slot"):
        c.check_status()
    ref = reference(c, 0, q, slots[:3] + [0], last)
    check(out, lse, ref)
    far = ip.clone(); far[2] = c.n_pages * P
    out, lse = c.decode_attention(0, q, bi, far, shared=g)
    with pytest.raises(RuntimeError, match="bad position"):
        c.check_status()
    check(out, lse, reference(c, 0, q, slots[:2] + [0, slots[3]], last))
    # a page in the middle of row 2 that is not mapped: its keys are not visible
    page = c.page_table[slots[2], 0].item()
    c._page_table[slots[2], 0] = -1
    out, lse = c.decode_attention(0, q, bi, ip, shared=g)
    c.check_status()
    plain, plain_lse = c.decode_attention(0, q, bi, ip)
    ref = reference(c, 0, q, slots, last)
    check(out[[0, 1, 3]], lse[[0, 1, 3]], [r[[0, 1, 3]] for r in ref])
    assert (out[2].double() - plain[2].double()).abs().max() <= 2.0 ** -7 * plain[2].abs().max() and (lse[2] - plain_lse[2]).abs().max() < 1e-5
    c._page_table[slots[2], 0] = page


@pytest.mark.parametrize("kw", [dict(dtype=torch.float32), dict(page_size=64), dict(Hq=34, Hkv=2)],
                         ids=["fp32", "page-64", "wide-heads"])
def test_shapes_served_row_by_row(kw):
    a = dict(Hq=4, Hkv=2, D=64, dtype=torch.bfloat16, page_size=128) | kw
    c, slots, last, q = build(a["Hq"], a["Hkv"], a["D"], a["dtype"], [(2, [300, 301])], (200,), page_size=a["page_size"])
    out, lse, _ = run(c, slots, last, q)
    ref = list(reference(c, 0, q, slots, last))
    check(out, lse, ref)


def test_captured_and_refilled():
    """A captured call follows its index tensors: other positions, another grouping, on the same addresses."""
    c, slots, last, q = build(16, 8, 128, torch.bfloat16, [(3, [500, 600, 700]), (2, [300, 301, 302])], ())
    n = len(slots)
    bi, ip = torch.tensor(slots, device="cuda"), torch.tensor(last, dtype=torch.int32, device="cuda")
    g = c.prefix_groups(slots)
    c.decode_attention(0, q, bi, ip, shared=g)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = c.decode_attention(0, q, bi, ip, shared=g)
        graphs.append((graph, got))
    order = [4, 5, 3, 1, 0, 2]
    for rows in (list(range(n)), order):
        s, p = [slots[i] for i in rows], [last[i] - 7 * (rows is order) for i in rows]
        bi.copy_(torch.tensor(s)); ip.copy_(torch.tensor(p))
        c.prefix_groups(s, into=g)
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        torch.cuda.synchronize()
        for (graph, _), st in zip(graphs, streams):      # side by side: every captured call has scratch of its own
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        c.check_status()
        ref = reference(c, 0, q, s, p)
        for _, (out, lse) in graphs:
            check(out, lse, ref)


def test_two_calls_are_the_same_bits():
    c, slots, last, q = build(16, 8, 128, torch.bfloat16, *BATCHES["very wide group"])
    a, la, _ = run(c, slots, last, q)
    b, lb, _ = run(c, slots, last, q, pos_dtype=torch.int64)
    assert torch.equal(a, b) and torch.equal(la, lb)


def test_device_tables_follow_shares_and_erases():
    """The device's stacks and tables equal the host's lists through shares, chains of them and erases in any order."""
    import random
    rng = random.Random(5)
    c = PagedKVCache(64, 128, 12, 1, 64, 1, torch.bfloat16, "cuda")
    held = {}
    for step in range(400):
        what = rng.choice(["new", "share", "grow", "erase"])
        if what == "new" and c.free_batch_idx:
            held[c.allocate()] = 0
        elif what == "share" and held and c.free_batch_idx:
            src = rng.choice(list(held)); n = rng.randint(0, len(c.page_table_cpu[src]))
            held[c.share_prefix(src, n * 128)] = 0
        elif what == "grow" and held:
            s = rng.choice(list(held)); want = (len(c.page_table_cpu[s]) + rng.randint(0, 4)) * 128
            if c.can_reserve(want, s):
                c.reserve(s, None, want)
        elif what == "erase" and held:
            s = rng.choice(list(held)); c.erase(s); del held[s]
        if rng.random() < 0.1 or step == 399:
            pt, il = c.page_table.cpu(), c.physical_to_logical.cpu()
            for s in range(1, 12):
                pages = c.page_table_cpu[s]
                assert pt[s, :len(pages)].tolist() == pages and (pt[s, len(pages):] == -1).all()
                assert {int(p): int(il[s, p]) for p in (il[s] >= 0).nonzero()} == {p: i for i, p in enumerate(pages)}
            np_, ns = c._alloc_counts.tolist()
            assert c._free_pages_dev[:np_].tolist() == c.free_pages and c._free_slots_dev[:ns].tolist() == c.free_batch_idx
            c.check_status()


@pytest.mark.parametrize("pages,rows,alone", [(63, 4, 3), (64, 4, 3), (65, 2, 1), (131, 3, 0), (190, 1, 2)])
def test_few_long_segments(pages, rows, alone):
    """So few segments that an even share would cut each into more pieces than the bound: one stored head, long single rows."""
    n = pages * P
    c, slots, last, q = build(8, 1, 128, torch.bfloat16, [(pages, [n + 1 + 37 * i for i in range(rows)])],
                              [n - 5 - 211 * i for i in range(alone)], seed=pages)
    out, lse, _ = run(c, slots, last, q)
    check(out, lse, reference(c, 0, q, slots, last))


@pytest.mark.parametrize("how", ["padding", "erased", "out of range"])
@pytest.mark.parametrize("rows,gone", [(4, [0]), (4, [0, 1, 2]), (4, [2]), (3, [0, 1, 2]), (70, list(range(40)))],
                         ids=["first", "all but the last", "middle", "all", "more than a warp looks at"])
def test_rows_that_have_ended(how, rows, gone):
    """Rows of a group whose request ended after the groups were made: nothing for them, whichever they are, and the others keep the
    prefix, also where it was named by one that has ended."""
    c, slots, last, q = build(4, 2, 64, torch.bfloat16, [(3, [390 + i for i in range(rows)]), (1, [200, 201])], (300,), seed=rows)
    g = c.prefix_groups(slots)
    want = [0 if b in gone else s for b, s in enumerate(slots)]
    if how == "erased":
        for b in gone:
            c.erase(slots[b])
        now = slots
    else:
        now = [s if b not in gone else (0 if how == "padding" else c.max_batch_size + b) for b, s in enumerate(slots)]
    bi, ip = torch.tensor(now, device="cuda"), torch.tensor(last, dtype=torch.int32, device="cuda")
    out, lse = c.decode_attention(0, q, bi, ip, shared=g)
    if how == "out of range":
        with pytest.raises(RuntimeError, match="bad slot"):
            c.check_status()
    c.check_status()
    check(out, lse, reference(c, 0, q, want, last), how)


@pytest.mark.parametrize("n", [100, 128, 1000])
def test_groups_with_common_rows_stay_inside_the_workspace(n):
    """Every group names all rows: two query tiles each, twice as many in all as the workspace has room for."""
    c, slots, last, q = build(4, 2, 64, torch.bfloat16, [(2, [257 + i for i in range(100)])], ())
    B, H = 100, 2
    bi, ip = torch.tensor(slots, device="cuda"), torch.tensor(last, dtype=torch.int32, device="cuda")
    groups = torch.tensor([[0, B, 2, 0]] * n, dtype=torch.int32, device="cuda")
    row_group = torch.zeros(B, dtype=torch.int32, device="cuda")
    out, lse = torch.empty(B, 4, 1, 64, dtype=q.dtype, device="cuda"), torch.empty(B, 4, 1, device="cuda")
    c.flush_tables()
    need = ctypes.c_size_t(0)
    assert _lib.lib.fpkv_decode_shared_workspace_bytes(ctypes.byref(c._pool), B, 4, n, ctypes.byref(need)) == 0
    behind = 64 << 20                                    # more than all the tiles named could write
    ws = torch.full((need.value + behind,), 0x5a, dtype=torch.uint8, device="cuda")
    rc = _lib.lib.fpkv_decode_attn_shared(ctypes.byref(c._pool), 0, out.data_ptr(), lse.data_ptr(), q.data_ptr(), q.stride(0), q.stride(1),
                                          bi.data_ptr(), ip.data_ptr(), _lib.FPKV_I32, B, 4, groups.data_ptr(), n, row_group.data_ptr(),
                                          0.125, ws.data_ptr(), need.value, None, c._status.data_ptr(),
                                          torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    torch.cuda.synchronize()
    assert (ws[need.value:] == 0x5a).all()
    with pytest.raises(RuntimeError, match="bad slot"):
        c.check_status()
    check(out, lse, reference(c, 0, q, slots, last, 0.125))          # their group is the first one, which fits


def test_records_of_another_form_are_refused():
    c, slots, last, q = build(4, 2, 64, torch.bfloat16, [(2, [300, 301, 302])], ())
    bi, ip = torch.tensor(slots, device="cuda"), torch.tensor(last, dtype=torch.int32, device="cuda")
    for groups, row_group in ((torch.zeros(1, 3), torch.zeros(3)), (torch.zeros(4), torch.zeros(3)), (torch.zeros(2, 5)[:, :4], torch.zeros(3)),
                              (torch.zeros(1, 4), torch.zeros(4)), (torch.zeros(1, 4), torch.zeros(6)[::2])):
        g = c.prefix_groups(slots)
        g.groups, g.row_group = (t.to(torch.int32).cuda() if t.is_contiguous() else torch.empty_strided(t.shape, t.stride(), dtype=torch.int32, device="cuda")
                                 for t in (groups, row_group))
        with pytest.raises(AssertionError):
            c.decode_attention(0, q, bi, ip, shared=g)
    g = c.prefix_groups(slots)
    for name, t in (("groups", g.groups.cpu()), ("row_group", g.row_group.cpu()), ("groups", g.groups.long()), ("row_group", g.row_group.long())):
        h = c.prefix_groups(slots)
        setattr(h, name, t)
        with pytest.raises(AssertionError):
            c.decode_attention(0, q, bi, ip, shared=h)
