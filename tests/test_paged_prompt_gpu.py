"""qmtp.paged.prompt_attention against the 64-bit reference, and append, prompt and decode run together."""
import pytest
import torch

from tests._paged_ref import BF16, Batch, attention_ref, check, visible

pytestmark = pytest.mark.gpu


def no_error():
    from qmtp import _lib

    torch.cuda.synchronize()
    assert _lib.device_error() == 0


def prompt(bt, **kw):
    from qmtp import paged

    gate = bt.d["gate"][:, :, 1] if kw.pop("gate", True) else None
    return paged.prompt_attention(*bt.args(), bt.d["cu"], gate=gate, **kw)


LAYOUTS = [(16, 4, 256, 64), (4, 2, 256, 16), (8, 1, 256, 256), (32, 8, 128, 16), (7, 1, 128, 32), (12, 12, 64, 128),
           (40, 2, 64, 256), (64, 1, 128, 64)]


@pytest.mark.parametrize("nq,nkv,dh,page", LAYOUTS)
def test_prompt_small(nq, nkv, dh, page, dev):
    bt = Batch([(5, 5)], nq, nkv, dh, page, seed=dh).put(dev)
    out = prompt(bt, gate=False)
    no_error()
    check(out, attention_ref(bt, gate=False))


@pytest.mark.parametrize("nq,nkv,dh,page", LAYOUTS)
def test_prompt_ragged(nq, nkv, dh, page, dev):
    """Chunks of one token and of several tiles, with and without earlier tokens, no tokens, an empty sequence
    and one that is shorter than its chunk."""
    bt = Batch([(1, 1), (33, 33), (0, 40), (130, 129 + 128), (3, 0), (5, 2), (65, 400), (1, 257), (128, 128)], nq, nkv, dh,
               page, seed=nq).put(dev)
    out = prompt(bt)
    no_error()
    check(out, attention_ref(bt))


@pytest.mark.parametrize("dh,nq,nkv", [(256, 4, 1), (128, 4, 2), (64, 3, 3)])
@pytest.mark.parametrize("n,length", [(700, 700), (1, 4000), (64, 2500), (300, 1111)])
def test_prompt_long(dh, nq, nkv, n, length, dev):
    bt = Batch([(n, length)], nq, nkv, dh, 64, seed=length).put(dev)
    out = prompt(bt)
    no_error()
    check(out, attention_ref(bt))


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 2), (64, 0), (100, 4), (128, 130), (257, 300), (1000, 4),
                                          (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("dh,nq,nkv,page", [(256, 4, 1, 32), (128, 10, 2, 16)])
def test_prompt_window(window, sinks, dh, nq, nkv, page, dev):
    bt = Batch([(150, 700), (40, 40), (9, 1200)], nq, nkv, dh, page, seed=window % 1000).put(dev)
    out = prompt(bt, window=window, sinks=sinks, scale=0.2)
    no_error()
    check(out, attention_ref(bt, window, sinks, scale=0.2))


@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 3)])
@pytest.mark.parametrize("poison", [float("nan"), float("-inf"), torch.finfo(BF16).min])
@pytest.mark.parametrize("dh", [256, 128])
def test_prompt_masked_places_hold_anything(window, sinks, poison, dh, dev):
    bt = Batch([(3, 3), (20, 20), (7, 130), (40, 333)], 8, 2, dh, 16, seed=3, table_extra=2)
    ref = attention_ref(bt, window, sinks)
    seen = torch.zeros(bt.pages, bt.page, dtype=torch.bool)
    need = torch.zeros_like(bt.table, dtype=torch.bool)
    for b, (n, length) in enumerate(bt.sizes):
        for p in range(length - n, length):
            keys = torch.tensor(visible(p, window, sinks))
            pg, sl = bt.rows(b, keys)
            seen[pg, sl] = True
            need[b, keys // bt.page] = True
    for t in (bt.k, bt.v):
        t.transpose(1, 2)[~seen] = poison
    bt.table[~need] = -1
    bt.put(dev)
    out = prompt(bt, window=window, sinks=sinks)
    no_error()
    check(out, ref)
    # a later token's own key and value: the earlier tokens of the chunk do not see them
    pg, sl = bt.rows(3, 320)
    bt.cache.v[pg, :, sl] = poison
    bt.cache.k[pg, :, sl] = poison
    out = prompt(bt, window=window, sinks=sinks)
    no_error()
    check(out, ref, rows=list(range(3 + 20 + 7 + 27)))


def test_prompt_growing_scores(dev):
    """Scores that rise by far more than the rescaling slack from key tile to key tile, and fall again."""
    for dh, nq in ((256, 2), (64, 2)):
        bt = Batch([(200, 900)], nq, 1, dh, 64, seed=dh)
        level = torch.cat([torch.linspace(0, 6, 600), torch.linspace(6, -6, 300)])
        pg, sl = bt.rows(0, torch.arange(900))
        bt.k[pg, :, sl, 0] = (level[:, None] * 8).to(BF16)
        bt.q[:, :, 0] = 8.0
        bt.put(dev)
        out = prompt(bt)
        no_error()
        check(out, attention_ref(bt))


def test_prompt_leaves_rows_of_no_sequence(dev):
    from qmtp import paged

    for dh in (256, 128):
        bt = Batch([(4, 10), (30, 44)], 4, 2, dh, 16, seed=2).put(dev)
        ref = attention_ref(bt, gate=False)
        q = torch.zeros((50, 4, dh), dtype=BF16, device=dev)
        q[7:41] = bt.d["q"]
        out = torch.full((50, 4 * dh), 3.0, dtype=BF16, device=dev)
        paged.prompt_attention(q, bt.cache, bt.d["table"], bt.d["lens"], bt.d["cu"] + 7, out=out)
        no_error()
        assert (out[:7] == 3).all() and (out[41:] == 3).all()
        check(out[7:41], ref)


def test_prompt_device_checks(dev):
    """A bad page reads as zeros, a bad length as an empty sequence, bad row offsets as no rows."""
    from qmtp import _lib

    bt = Batch([(20, 40), (20, 40)], 2, 1, 128, 16, seed=6).put(dev)
    good = prompt(bt)
    no_error()

    def bad():
        out = prompt(bt)
        torch.cuda.synchronize()
        assert _lib.device_error() == 2
        return out

    for value in (bt.pages, -1, 2 ** 31 - 1):
        bt.d["table"][0, 1] = value
        out = bad()
        assert torch.isfinite(out).all() and torch.equal(out[20:], good[20:])
    for value in (49, -1, 2 ** 31 - 1):
        bt.d["lens"][0] = value
        out = bad()
        assert (out[:20] == 0).all() and torch.equal(out[20:], good[20:])
    bt = Batch([(20, 40), (20, 40)], 2, 1, 128, 16, seed=6).put(dev)
    for value in (41, 2 ** 31 - 1, -1):
        bt.d["cu"][2] = value
        assert torch.equal(bad()[:20], good[:20])


@pytest.mark.parametrize("dh,nq,nkv,window", [(256, 16, 4, 0), (128, 10, 2, 70), (64, 4, 4, 0)])
def test_serving_run(dh, nq, nkv, window, dev):
    """As a serving loop runs them: prompts appended and attended in chunks, then verify steps of 3 tokens of
    which some are kept, all against one pass over the final keys."""
    from qmtp import paged

    g = torch.Generator().manual_seed(dh)
    lengths, page, sinks = [150, 37, 260], 16, 3 if window else 0
    total = [n + 12 for n in lengths]
    width = (2 * nq + 2 * nkv) * dh
    x = [torch.randn((n, width), generator=g).to(BF16) for n in total]
    qn, kn = ((1 + 0.2 * torch.randn(dh, generator=g)).to(BF16).to(dev) for _ in range(2))
    rot = 32
    ang = torch.arange(400)[:, None] * 1e4 ** (-torch.arange(rot // 2) / (rot // 2))
    kw = dict(n_heads=nq, gated=True, q_norm=qn, k_norm=kn, cos=ang.cos().to(dev), sin=ang.sin().to(dev))
    pages = sum(-(-n // page) for n in total)
    table = torch.full((3, max(-(-n // page) for n in total)), -1, dtype=torch.int32)
    order, at = torch.randperm(pages, generator=g).to(torch.int32), 0
    for b, n in enumerate(total):
        table[b, : -(-n // page)] = order[at: at + -(-n // page)]
        at += -(-n // page)
    table = table.to(dev)
    cache = paged.PagedCache.empty(pages, nkv, dh, page, dev)
    cache.k.fill_(float("nan"))
    cache.v.fill_(float("nan"))
    got = [[] for _ in total]
    done = [0, 0, 0]

    def rows(new):
        return torch.cat([x[b][done[b]: done[b] + n] for b, n in enumerate(new)]).to(dev)

    while any(d < n for d, n in zip(done, lengths)):  # prompts, at most 100 tokens a chunk
        new = [min(100, n - d) for d, n in zip(done, lengths)]
        lens = torch.tensor([d + n for d, n in zip(done, new)], dtype=torch.int32, device=dev)
        cu = torch.tensor([0, *torch.tensor(new).cumsum(0)], dtype=torch.int32, device=dev)
        q, gate = paged.append_qkv(rows(new), cache, table, lens, cu, **kw)
        out = paged.prompt_attention(q, cache, table, lens, cu, gate=gate, window=window, sinks=sinks).cpu()
        for b, o in enumerate(out.split(new)):
            got[b].append(o)
        done = [d + n for d, n in zip(done, new)]
    for keep in (1, 3, 2, 3, 1, 2):  # 12 tokens
        new = [3, 3, 3]
        xs = torch.cat([torch.cat([x[b][done[b]: done[b] + keep], torch.randn((3 - keep, width), generator=g).to(BF16)])
                        for b in range(3)]).to(dev)
        lens = torch.tensor([min(d + 3, n) for d, n in zip(done, total)], dtype=torch.int32, device=dev)
        short = [int(d + 3 - n) for d, n in zip(done, lens.tolist())]  # the last steps end with the table
        if any(short):
            xs = torch.cat([x[b][done[b] - short[b]: done[b] - short[b] + 3] for b in range(3)]).to(dev)
        q, gate = paged.append_qkv(xs, cache, table, lens, **kw)
        out = paged.attention(q, cache, table, lens, gate=gate, window=window, sinks=sinks).cpu()
        for b in range(3):
            got[b].append(out[3 * b + short[b]: 3 * b + short[b] + keep])
        done = [d + keep for d in done]
    no_error()
    assert done == total
    # one pass: the same norms and rotation, then the reference
    bt = Batch([(n, n) for n in total], nq, nkv, dh, page, seed=1)
    bt.table[:] = table.cpu()[:, : bt.table.shape[1]].clamp_min(0)
    bt.k, bt.v = torch.zeros((pages, nkv, page, dh), dtype=BF16), torch.zeros((pages, nkv, page, dh), dtype=BF16)
    bt.put(dev)
    q, gate = paged.append_qkv(torch.cat(x).to(dev), bt.cache, bt.d["table"], bt.d["lens"], bt.d["cu"], **kw)
    no_error()
    bt.q, bt.k, bt.v = q.cpu(), bt.cache.k.cpu(), bt.cache.v.cpu()
    bt.gate = torch.stack([gate.cpu(), gate.cpu()], 2)
    check(torch.cat([torch.cat(o) for o in got]), attention_ref(bt, window, sinks))


def test_prompt_in_a_graph(dev):
    """A captured chunk replayed over other lengths and rows, against eager calls; two graphs, one workspace pool."""
    bt = Batch([(60, 200), (9, 77)], 16, 4, 256, 64, seed=11).put(dev)
    prompt(bt)
    torch.cuda.synchronize()
    a, b = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(a):
        oa = prompt(bt)
    with torch.cuda.graph(b, pool=a.pool()):
        ob = prompt(bt, window=40, sinks=2)
    for lens in ([200, 77], [60, 9], [130, 100]):
        bt.d["lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        a.replay()
        b.replay()
        assert torch.equal(oa, prompt(bt)) and torch.equal(ob, prompt(bt, window=40, sinks=2))
    no_error()


@pytest.mark.parametrize("nq,nkv,dh", [(4, 1, 256), (6, 2, 128), (2, 2, 64)])
def test_prompt_many_short_sequences(nq, nkv, dh, dev):
    """More items than SMs, a few keys each, so that every block works through many of them one behind the other:
    one token, chunks that fill one row tile or two, a sequence end in every item."""
    sizes = [(1 + (i * 7) % 90, 1 + (i * 7) % 90 + (i * 5) % 140) for i in range(250)]
    bt = Batch(sizes, nq, nkv, dh, 16, seed=dh).put(dev)
    out = prompt(bt)
    no_error()
    check(out, attention_ref(bt))
    for _ in range(5):
        assert torch.equal(prompt(bt), out)
    no_error()


def test_pool_beyond_32_bit_offsets(dev):
    """Pages whose elements lie beyond 2^31 from the pool's start: append, decode and prompt attention there."""
    from qmtp import paged

    small = Batch([(3, 200), (3, 70)], 4, 2, 256, 64, seed=21)
    pages = 2 ** 31 // (2 * 64 * 256) + 40
    cache = paged.PagedCache.empty(pages, 2, 256, 64, dev)
    first = pages - small.pages
    cache.k[first:], cache.v[first:] = small.k.to(dev), small.v.to(dev)
    small.put(dev)
    table = small.d["table"] + first
    q, lens, cu = small.d["q"], small.d["lens"], small.d["cu"]
    assert torch.equal(paged.attention(q, cache, table, lens), paged.attention(*small.args()))
    assert torch.equal(paged.prompt_attention(q, cache, table, lens, cu), paged.prompt_attention(*small.args(), cu))
    qkv = torch.randn((6, 8 * 256), device=dev).to(BF16)
    for c, t in ((cache, table), (small.cache, small.d["table"])):
        paged.append_qkv(qkv, c, t, lens, n_heads=4)
    no_error()
    assert torch.equal(cache.k[first:], small.cache.k) and torch.equal(cache.v[first:], small.cache.v)
