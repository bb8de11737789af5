"""GPU: packed-row indices, block tables and slot maps from device-held request lengths, against plain loops; and the
whole serving step: tables -> append -> prefill, shared prefixes -> decode -> sampling."""

import pytest
import torch

from fpkv.engine_glue import SlotState, PrefillChunk, pack_prefill_rows
from fpkv.paged_attention import PagedKVCache

pytestmark = pytest.mark.gpu


def loops(c, slots, starts, lens, L, W, align, tokens, pad):
    P = c.page_size
    table = c.page_table.cpu()
    ids, pos, bi, row = [pad] * L, [0] * L, [0] * L, [-1] * L
    offsets, last, at, k = [], [], 0, 0
    for s, a, n in zip(slots, starts, lens):
        offsets.append(at)
        for i in range(n):
            if at + i < L and s > 0:
                p = a + i
                ids[at + i], pos[at + i], bi[at + i] = tokens[k + i], p, s
                pg = int(table[s, p // P]) if p // P < c.n_pages else -1
                row[at + i] = pg * P + p % P if pg >= 0 else -1
        last.append(at + n - 1 if n and at + n <= L else -1)
        at += -(-n // align) * align
        k += n
    block = [[int(table[s, j]) if s > 0 and j * P < a + n and j < c.n_pages else -1 for j in range(W)] for s, a, n in zip(slots, starts, lens)]
    return ids, pos, bi, row, block, [a + n for a, n in zip(starts, lens)], offsets + [at], last


def cache_for(need, page_size=128, seed=0, extra=2):
    pages = [-(-n // page_size) for n in need]
    c = PagedKVCache(1 + sum(pages) + extra, page_size, len(need) + 2, 1, 64, 1, torch.bfloat16, "cuda")
    c.free_pages = (torch.randperm(c.n_pages - 1, generator=torch.Generator().manual_seed(seed)) + 1).tolist()
    slots = []
    for n in need:
        slots.append(c.allocate()); c.reserve(slots[-1], None, n)
    return c, slots


def dev(x, t):
    return torch.tensor(x, dtype=t, device="cuda")


def check(c, slots, starts, lens, L, W=None, align=128, pad=0, with_tokens=True):
    tokens = [1000 + i for i in range(sum(lens))]
    t = c.step_tables(dev(slots, torch.int64), dev(starts, torch.int32), dev(lens, torch.int32), L, W, align,
                      dev(tokens, torch.int64) if with_tokens else None, pad)
    W = c.n_pages if W is None else W
    ids, pos, bi, row, block, seq, off, last = loops(c, slots, starts, lens, L, W, align, tokens, pad)
    assert t.input_pos.shape == t.batch_idx.shape == (1, L) and t.pool_row.shape == (L,) and t.block_table.shape == (len(slots), W)
    assert (t.input_ids is None) == (not with_tokens)
    if with_tokens:
        assert t.input_ids[0].tolist() == ids
    assert t.input_pos[0].tolist() == pos and t.batch_idx[0].tolist() == bi and t.pool_row.tolist() == row
    assert t.block_table.tolist() == block and t.seq_lens.tolist() == seq and t.offsets.tolist() == off and t.last.tolist() == last


@pytest.mark.parametrize("lens,starts", [([1], [0]), ([1, 1, 1], [5, 0, 127]), ([0, 3, 0, 0, 130, 0], [0, 126, 9, 0, 0, 0]),
                                         ([128, 256, 129], [0, 0, 128]), ([700, 1, 33, 5], [1, 511, 100, 1023]), ([0, 0], [0, 3])])
@pytest.mark.parametrize("align", [1, 16, 128])
@pytest.mark.parametrize("page_size", [16, 128])
def test_against_loops(lens, starts, align, page_size):
    c, slots = cache_for([max(1, a + n) for a, n in zip(starts, lens)], page_size)
    used = sum(-(-n // align) * align for n in lens)
    for L in (used, used + 1, used + 333):
        check(c, slots, starts, lens, L, align=align, pad=-7)
    check(c, slots, starts, lens, used, W=0, align=align, with_tokens=False)
    check(c, slots, starts, lens, used, W=3, align=align)
    c.check_status()


@pytest.mark.parametrize("N", [255, 256, 257, 1000, 4096])
def test_many_requests(N):
    gen = torch.Generator().manual_seed(N)
    lens = torch.randint(0, 20, (N,), generator=gen).tolist()
    starts = torch.randint(0, 200, (N,), generator=gen).tolist()
    c, slots = cache_for([max(1, a + n) for a, n in zip(starts, lens)])
    check(c, slots, starts, lens, sum(-(-n // 16) * 16 for n in lens) + 5, W=2, align=16)
    c.check_status()


def test_no_requests_and_no_row():
    c, slots = cache_for([10])
    check(c, [], [], [], 40)
    check(c, [], [], [], 0)
    check(c, slots, [0], [0], 0)
    c.check_status()


def test_overflow_padding_and_bad_requests():
    c, slots = cache_for([300, 300, 300])
    status = lambda what: pytest.raises(RuntimeError, match=what)
    check(c, slots, [0, 0, 0], [100, 100, 100], 250, align=16)                 # the last request does not fit
    with status("bad position"):
        c.check_status()
    check(c, [slots[0], 0, slots[2]], [0, 0, 7], [20, 30, 10], 200, align=16)  # slot 0: a bucket's padding request
    c.check_status()
    i32, i64 = torch.int32, torch.int64
    t = c.step_tables(dev([slots[0], 99, slots[2]], i64), dev([0, 0, 0], i32), dev([5, 6, 7], i32), 64, 2, 16)
    with status("bad slot"):
        c.check_status()
    assert t.batch_idx[0, 16:32].tolist() == [0] * 16 and (t.block_table[1] == -1).all() and t.batch_idx[0, 32:39].tolist() == [slots[2]] * 7
    t = c.step_tables(dev(slots, i64), dev([0, -1, 0], i32), dev([5, 6, -7], i32), 64, 2, 16)
    with status("bad position"):
        c.check_status()
    assert t.offsets.tolist() == [0, 16, 16, 16] and t.last.tolist() == [4, -1, -1] and t.batch_idx.ne(0).sum() == 5
    t = c.step_tables(dev(slots[:1], i64), dev([380], i32), dev([10], i32), 16, 2, 16)      # four tokens past the reserved pages
    with status("bad page"):
        c.check_status()
    assert t.pool_row.ge(0).tolist() == [True] * 4 + [False] * 12 and t.batch_idx[0, :10].tolist() == [slots[0]] * 10
    t = c.step_tables(dev(slots[:1], i64), dev([c.n_pages * 128 - 2], i32), dev([4], i32), 16, 2, 16)
    with status("bad"):
        c.check_status()
    t = c.step_tables(dev(slots, i64), dev([0, 0, 0], i32), dev([2 ** 31 - 1] * 3, i32), 64, 0, 128)   # sums past 32 bits
    with status("bad position"):
        c.check_status()
    assert t.offsets.tolist() == [0] + [2 ** 31 - 1] * 3 and t.last.tolist() == [-1] * 3 and (t.batch_idx == slots[0]).all()
    c.step_tables(dev(slots, i64), dev([0, 0, 0], i32), dev([5, 5, 5], i32), 64, 2, 16, dev([1, 2, 3, 4, 5, 6], i64))
    with status("bad position"):
        c.check_status()


def test_same_row_as_the_host_packer():
    class Seq:
        def __init__(self, slot, n): self.batch_idx, self.total_length = slot, n
    c, slots = cache_for([400, 130, 1, 256])
    seqs = [Seq(s, n) for s, n in zip(slots, (400, 130, 1, 256))]
    chunks = [PrefillChunk(seqs[0], 128, 300), PrefillChunk(seqs[1], 0, 130), PrefillChunk(seqs[2], 0, 1), PrefillChunk(seqs[3], 255, 256)]
    ids = {id(s): torch.arange(s.total_length) + 10 * i for i, s in enumerate(seqs)}
    want = pack_prefill_rows(chunks, lambda s: ids[id(s)])
    t = c.step_tables(dev([ch.seq.batch_idx for ch in chunks], torch.int64), dev([ch.start for ch in chunks], torch.int32),
                      dev([ch.end - ch.start for ch in chunks], torch.int32), want[0].shape[1],
                      tokens=torch.cat([ids[id(ch.seq)][ch.start:ch.end] for ch in chunks]).cuda())
    assert torch.equal(t.input_ids.cpu(), want[0]) and torch.equal(t.input_pos.cpu(), want[1]) and torch.equal(t.batch_idx.cpu(), want[2])
    assert t.offsets[:-1].tolist() == want[3]


def test_captured_with_new_lengths():
    c, slots = cache_for([300, 300, 300])
    s, a, n = dev(slots, torch.int64), dev([0, 0, 0], torch.int32), dev([5, 6, 7], torch.int32)
    c.step_tables(s, a, n, 512)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        t = c.step_tables(s, a, n, 512)
    a.copy_(torch.tensor([10, 20, 30])); n.copy_(torch.tensor([129, 0, 1]))
    graph.replay()
    torch.cuda.synchronize()
    ids, pos, bi, row, block, seq, off, last = loops(c, slots, [10, 20, 30], [129, 0, 1], 512, c.n_pages, 128, [0] * 130, 0)
    assert t.input_pos[0].tolist() == pos and t.batch_idx[0].tolist() == bi and t.pool_row.tolist() == row
    assert t.block_table.tolist() == block and t.offsets.tolist() == off and t.last.tolist() == last and t.seq_lens.tolist() == seq


def test_a_serving_step_together():
    """Five questions about one picture: the picture prefilled once, its pages shared, the questions prefilled from tables
    built on the device, then decode steps with shared-prefix attention and sampling -- against the same requests served
    separately, each with pages of its own."""
    Hq, Hkv, D, V, P, dtype = 4, 2, 128, 500, 128, torch.bfloat16
    gen = torch.Generator(device="cuda").manual_seed(0)
    R = lambda *s: (torch.randn(*s, generator=gen, device="cuda") * 0.5).to(dtype)
    table = {"q": R(V, Hq, D), "k": R(V, Hkv, D), "v": R(V, Hkv, D)}       # a one-layer model: token -> q, k, v; output -> logits
    head = R(Hq * D, V)
    picture = torch.randint(1, V, (2 * P,), generator=gen, device="cuda")
    asks = [torch.randint(1, V, (n,), generator=gen, device="cuda") for n in (3, 40, 1, 130, 17)]
    uniform = torch.rand(6, len(asks), generator=gen, device="cuda")

    def prefill(c, slots, starts, lens, tokens):
        L = int(sum(-(-int(x) // P) * P for x in lens))
        t = c.step_tables(dev(slots, torch.int64), dev(starts, torch.int32), dev(lens, torch.int32), L, tokens=tokens)
        pick = lambda n: table[n][t.input_ids[0]].transpose(0, 1)[None]
        c.insert_kv(0, pick("k"), pick("v"), input_pos=t.input_pos, batch_idx=t.batch_idx)
        mask = c.create_prefill_blockmask(t.batch_idx, t.input_ids, V + 1, V + 2)
        out, _ = c.prefill_attention(0, pick("q"), t.batch_idx, t.input_pos, mask, token_major=True)
        return out[0, t.last.long()].reshape(len(lens), Hq * D), t

    def serve(shared):
        c = PagedKVCache(40, P, 8, Hkv, D, 1, dtype, "cuda")
        lens = [len(a) for a in asks]
        if shared:
            base = c.allocate(); c.reserve(base, None, 2 * P)
            prefill(c, [base], [0], [2 * P], picture)
            slots = [c.share_prefix(base, 2 * P) for _ in asks]
            for s, n in zip(slots, lens):
                c.reserve(s, None, 2 * P + n + 8)
            c.erase(base)                                # the questions hold the picture now
            h, _ = prefill(c, slots, [2 * P] * 5, lens, torch.cat(asks))
        else:
            slots = [c.allocate() for _ in asks]
            for s, n in zip(slots, lens):
                c.reserve(s, None, 2 * P + n + 8)
            h, _ = prefill(c, slots, [0] * 5, [2 * P + n for n in lens], torch.cat([torch.cat([picture, a]) for a in asks]))
        state, groups = SlotState(8, "cuda"), c.prefix_groups(slots, rows=6)
        assert groups.n_groups == (1 if shared else 0)
        logits, hidden = [], []
        from fpkv.sampling import sample
        tok, _ = sample(h @ head, uniform[0], temperature=0.7, top_k=40, top_p=0.95)
        for s, n, tk in zip(slots, lens, tok.tolist()):
            state.begin(s, 2 * P + n, 2 * P + n, tk)
        toks = [tok.tolist()]
        for step in range(1, 6):
            B = state.stage(slots, bucket=6)             # one padding row
            bi, ip, _, ids = state.step_inputs(B)
            pick = lambda n: table[n][ids][:, :, None]
            out, _ = c.decode_step(0, pick("q"), pick("k"), pick("v"), bi, ip, shared=groups)
            hidden.append(out[:5].float().cpu())
            u = torch.cat([uniform[step], uniform[step][:1]])
            tok, _ = state.sample(B, out.reshape(B, Hq * D) @ head, u, temperature=0.7, top_k=40, top_p=0.95)
            toks.append(tok[:5].tolist())
        c.check_status()
        for s in slots:
            c.erase(s)
        assert c.num_free_pages == 39
        return toks, hidden

    (ta, ha), (tb, hb) = serve(True), serve(False)
    # the two differ in roundings alone; once a token differs (a draw within those roundings of a border) so may the rest of its row
    for i in range(5):
        for step in range(6):
            if ta[step][i] != tb[step][i]:
                assert step > 0, "the prefills see the same keys in the same order"
                break
            if step < 5:
                assert (ha[step][i] - hb[step][i]).abs().max() <= 2.0 ** -6 * hb[step][i].abs().max()
    assert sum(a == b for a, b in zip(sum(ta, []), sum(tb, []))) >= 24


def test_rows_that_end_behind_the_last_token():
    """The last request's run need not fit, only its tokens; nor need a padding request, whose tokens are pads."""
    c, slots = cache_for([300, 300])
    for align in (16, 128):
        check(c, slots, [0, 7], [100, 33], -(-100 // align) * align + 33, align=align)
        check(c, slots[:1], [0], [5], 5, align=align)
        check(c, slots + [0], [0, 7, 0], [100, 33, 50], -(-100 // align) * align + 40, align=align)
        check(c, slots, [0, 7], [100, 0], 100, align=align)
    c.check_status()
    check(c, slots, [0, 7], [100, 33], 128 + 32)
    with pytest.raises(RuntimeError, match="bad position"):
        c.check_status()
    check(c, slots, [0, 7], [100, 33], 99)
    with pytest.raises(RuntimeError, match="bad position"):
        c.check_status()
