"""Edges of the paged-cache operators (qmtp.paged): optional arguments on their own, infinities and NaN in every
place, row offsets that are no offsets.  64-bit references and tolerances as in _paged_ref."""
import pytest
import torch

from tests._paged_ref import BF16, Batch, append_ref, attention_ref, check

pytestmark = pytest.mark.gpu


def device_error():
    from qmtp import _lib

    torch.cuda.synchronize()
    return _lib.device_error()


# ------------------------------------------------------------------------------------ append
@pytest.mark.parametrize("nq,nkv,dh,rotary,gated", [
    (7, 1, 128, 48, True), (5, 5, 64, 64, True), (3, 1, 64, 0, False), (16, 4, 256, 64, True), (6, 2, 64, 32, False)])
@pytest.mark.parametrize("norm", ["q", "k"])
@pytest.mark.parametrize("T", [5, 400, 9600])
def test_append_with_one_norm(nq, nkv, dh, rotary, gated, norm, T, dev):
    """A norm of the queries alone, and of the keys alone: a warp's step holds rows with a norm beside rows without one
    where the query heads do not fill it; by each of the ways that the kernel deals rows."""
    from qmtp import paged

    n = T // 5
    bt = Batch([(n, n + 3), (T - n, T - n + 17)], nq, nkv, dh, 32, seed=T + dh)
    width = (nq * (2 if gated else 1) + 2 * nkv) * dh
    qkv = torch.randn((T, width), generator=bt.g).to(BF16)
    w = (1 + 0.3 * torch.randn(dh, generator=bt.g)).to(BF16)
    qn, kn = (w, None) if norm == "q" else (None, w)
    cos = sin = None
    if rotary:
        ang = torch.arange(T + 20)[:, None] * 1e4 ** (-torch.arange(rotary // 2) / (rotary // 2))
        cos, sin = ang.cos().float(), ang.sin().float()
    rq, rqt, rk, rkt, rv = append_ref(bt, qkv, gated, qn, kn, cos, sin, 1e-6)
    bt.put(dev)
    dd = lambda t: None if t is None else t.to(dev)
    q, _ = paged.append_qkv(qkv.to(dev), bt.cache, bt.d["table"], bt.d["lens"], bt.d["cu"], n_heads=nq, gated=gated,
                            q_norm=dd(qn), k_norm=dd(kn), cos=dd(cos), sin=dd(sin))
    assert device_error() == 0
    assert ((q.cpu().double() - rq).abs() <= rqt).all()
    assert ((bt.cache.k.cpu().double() - rk).abs() <= rkt).all()
    assert torch.equal(bt.cache.v.cpu().double(), rv)


@pytest.mark.parametrize("spare", [0, 40])
@pytest.mark.parametrize("at,value", [(2, 3), (2, -1), (2, 30), (3, 31), (3, 2 ** 31 - 1), (0, -1), (1, 2 ** 31 - 1)])
def test_append_row_offsets_that_are_none(at, value, spare, dev):
    """Offsets that decrease or leave [0, rows] set the error word; the sequences they bound have no rows, the others keep
    theirs.  ``spare``: empty sequences before and behind, so that offsets fill more than one step of the search."""
    from qmtp import paged

    sizes = [(0, 5)] * spare + [(10, 20), (10, 20), (10, 20)] + [(0, 5)] * spare
    bt = Batch(sizes, 2, 1, 64, 16, seed=at)
    bt.cu[spare + at] = value
    want_k, want_v = bt.k.clone(), bt.v.clone()
    qkv = torch.randn((30, 4 * 64), generator=bt.g).to(BF16)
    want_q = torch.full((30, 2, 64), 3.0, dtype=BF16)
    offsets = bt.cu.tolist()
    holder = {}
    for b in reversed(range(len(sizes))):  # a row that two hold is the first one's
        c0, c1 = offsets[b], offsets[b + 1]
        if 0 <= c0 <= c1 <= 30:
            holder.update({t: (b, c1) for t in range(c0, c1)})
    for t, (b, c1) in holder.items():
        p = int(bt.lens[b]) - c1 + t
        if p >= 0:
            pg, sl = bt.rows(b, p)
            want_k[pg, 0, sl], want_v[pg, 0, sl], want_q[t] = qkv[t, 128:192], qkv[t, 192:], qkv[t, :128].view(2, 64)
    bt.put(dev)
    out = torch.full((30, 2, 64), 3.0, dtype=BF16, device=dev)
    paged.append_qkv(qkv.to(dev), bt.cache, bt.d["table"], bt.d["lens"], bt.d["cu"], n_heads=2, out=out)
    bad = any(not 0 <= c0 <= c1 <= 30 for c0, c1 in zip(offsets, offsets[1:]))  # 0, 10, 30, 30 are offsets
    assert device_error() == (2 if bad else 0)
    assert torch.equal(out.cpu(), want_q)
    assert torch.equal(bt.cache.k.cpu(), want_k) and torch.equal(bt.cache.v.cpu(), want_v)


# ------------------------------------------------------------------------------------ attention
def set_value(bt, b, pos, dim, value):
    """V of position pos of sequence b, every key head: value at dim."""
    pg, sl = bt.rows(b, pos)
    bt.v[pg, :, sl, dim] = value


@pytest.mark.parametrize("table_extra", [0, 200])
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dh", [256, 128, 64])
def test_prompt_rows_before_the_sequence_are_zeros(dh, poison, table_extra, dev):
    """A chunk longer than its sequence: its first rows see no key and give zeros, whatever the values in their tile are;
    with a wide table the keys are split and joined."""
    from qmtp import paged

    bt = Batch([(5, 2), (40, 33)], 4, 2, dh, 16, seed=dh, table_extra=table_extra)
    ref = attention_ref(bt)
    for b in range(2):
        set_value(bt, b, 0, 5, poison)
    bt.put(dev)
    out = paged.prompt_attention(*bt.args(), bt.d["cu"], gate=bt.d["gate"][:, :, 1]).cpu()
    assert device_error() == 0
    unseen = torch.tensor([True] * 3 + [False] * 2 + [True] * 7 + [False] * 33)
    assert (out[unseen] == 0).all()
    heads = out.view(-1, 4, dh)
    assert not torch.isfinite(heads[~unseen][..., 5]).any()
    rest = torch.arange(dh) != 5
    cut = lambda t: t.view(-1, 4, dh)[..., rest].reshape(t.shape[0], -1)
    check(cut(out), (cut(ref[0]), cut(ref[1])))


@pytest.mark.parametrize("dh,nq,nkv,S", [(64, 4, 2, 2), (128, 4, 2, 1), (256, 4, 2, 3)])
@pytest.mark.parametrize("length,window,sinks", [(100, 0, 0), (1000, 0, 0), (2048, 0, 0), (1500, 600, 300), (3500, 0, 0)])
def test_decode_infinite_value_in_any_slab(dh, nq, nkv, S, length, window, sinks, dev):
    """An infinite value that is seen gives an infinity in its dim and leaves the others, in whichever slab of keys it lies
    and by each form of the join, which agree bit for bit: in one launch (short tables), a block a row (few rows), a
    warp a row (many)."""
    from qmtp import paged

    bt = Batch([(S, length)], nq, nkv, dh, 64, seed=length + dh).put(dev)
    q, cache, table, lens = bt.args()
    wide = torch.full((1, 1000), -1, dtype=torch.int32, device=dev)
    wide[:, : table.shape[1]] = table
    many = 1 + 2 * 148 // (S * nq)
    kw = dict(window=window, sinks=sinks)
    seen = [j for j in range(0, length - S + 1, 128) if not window or j < sinks or length - S - j < window] + [length - S]
    for j in seen:
        pg, sl = bt.rows(0, j)
        for value in (float("inf"), float("-inf")):
            held = cache.v[pg, :, sl, 5].clone()
            cache.v[pg, :, sl, 5] = value
            short = paged.attention(q, cache, table, lens, **kw)
            block = paged.attention(q, cache, wide, lens, **kw)
            warp = paged.attention(q.repeat(many, 1, 1), cache, wide.repeat(many, 1), lens.repeat(many), **kw)
            cache.v[pg, :, sl, 5] = held
            heads = short.view(S, nq, dh)
            assert (heads[..., 5] == value).all(), (j, value)
            assert torch.isfinite(heads[..., :5]).all() and torch.isfinite(heads[..., 6:]).all(), (j, value)
            assert torch.equal(short, block) and torch.equal(warp, block.repeat(many, 1)), (j, value)
    assert device_error() == 0


@pytest.mark.parametrize("nq,nkv,dh", [(16, 4, 256), (8, 4, 128), (4, 4, 64)])
def test_prompt_call_with_far_more_places_than_rows(nq, nkv, dh, dev):
    """Most of q's rows belong to no sequence and most sequences have no new token: the blocks' places without rows lie
    between, before and behind those with rows."""
    from qmtp import paged

    sizes = [(0, 3)] * 70 + [(90, 90)] + [(0, 0)] * 60 + [(1, 200), (130, 400)] + [(0, 1)] * 100 + [(33, 30), (0, 9)]
    bt = Batch(sizes, nq, nkv, dh, 16, seed=dh).put(dev)
    ref = attention_ref(bt, gate=False)
    T, first = 20000, 12345
    q = torch.full((T, nq, dh), float("nan"), dtype=BF16, device=dev)
    q[first: first + bt.T] = bt.d["q"]
    for _ in range(3):
        out = torch.full((T, nq * dh), 3.0, dtype=BF16, device=dev)
        paged.prompt_attention(q, bt.cache, bt.d["table"], bt.d["lens"], bt.d["cu"] + first, out=out)
        assert device_error() == 0
        assert (out[:first] == 3).all() and (out[first + bt.T:] == 3).all()
        check(out[first: first + bt.T], ref)


@pytest.mark.parametrize("table_extra", [0, 300])
@pytest.mark.parametrize("dh,nq,nkv,copies", [(64, 4, 2, 1), (128, 4, 2, 1), (256, 4, 2, 1), (64, 4, 2, 60), (256, 4, 2, 60)])
def test_scores_of_minus_infinity(dh, nq, nkv, copies, table_extra, dev):
    """A key whose score is -inf has weight 0; a query that sees only such keys has no softmax (0 / 0) and gives NaN, as the
    definition does, while one that sees no key gives zeros."""
    from qmtp import paged

    S = 3
    sizes = [(S, 1), (S, 2), (S, 500), (S, 300)] * copies
    bt = Batch(sizes, nq, nkv, dh, 16, seed=dh, table_extra=table_extra)
    bt.q[:, :, 0] = 1.0
    for b, (_, length) in enumerate(bt.sizes):
        pg, sl = bt.rows(b, torch.arange(length if b % 4 == 3 else 1))
        bt.k[pg, :, sl, 0] = float("-inf")
    ref = attention_ref(bt, gate=False)
    bt.put(dev)
    # sequence 0 sees its one key, sequence 1 that key and then a second one, 2 four hundred others, 3 only such keys
    kind = torch.tensor([0, 0, 1, 0, 1, 2, 2, 2, 2, 1, 1, 1] * copies)  # 0: no key, 1: NaN, 2: the reference
    for out in (paged.attention(*bt.args()), paged.prompt_attention(*bt.args(), bt.d["cu"])):
        out = out.cpu()
        assert (out[kind == 0] == 0).all() and torch.isnan(out[kind == 1]).all()
        check(out, ref, rows=kind == 2)
    assert device_error() == 0


@pytest.mark.parametrize("nq,nkv,dh", [(4, 1, 256), (6, 2, 128), (8, 2, 128), (2, 2, 64)])
def test_prompt_lone_and_paired_row_tiles_in_turn(nq, nkv, dh, dev):
    """Chunks of one row tile and of two follow one another in every block, a few key tiles each: the same bits every time,
    with what the kernel reads in the caches and not, and those of each sequence by itself."""
    from qmtp import paged

    sizes = [(1 + (i * 7) % 90, 1 + (i * 7) % 90 + (i * 5) % 140) for i in range(250)]
    bt = Batch(sizes, nq, nkv, dh, 16, seed=dh).put(dev)
    flush = torch.empty(64 << 20, dtype=torch.int32, device=dev)
    alone = [paged.prompt_attention(bt.d["q"][c:c + n], bt.cache, bt.d["table"][b:b + 1], bt.d["lens"][b:b + 1],
                                    torch.tensor([0, n], dtype=torch.int32, device=dev))
             for b, ((n, _), c) in enumerate(zip(sizes, bt.cu.tolist()))]
    alone = torch.cat(alone)
    wrong = torch.zeros(300, dtype=torch.bool, device=dev)
    for i in range(300):
        if i % 3 == 0:
            flush.fill_(i)
        wrong[i] = (paged.prompt_attention(*bt.args(), bt.d["cu"]) != alone).any()
    assert device_error() == 0
    assert not wrong.any(), int(wrong.sum())
def check_classes(out, ref, bt, marks, window=0, sinks=0, gate=None):
    """out against ref in every (row, dim) whose seen values are finite; in the others the infinity or NaN that the seen
    marks (sequence, position, dim, value) add up to."""
    out = out.cpu().view(bt.T, bt.nq, bt.dh)
    r, kind = 0, torch.zeros(bt.T, bt.dh, dtype=torch.long)  # bits: inf 1, -inf 2, NaN 4
    for b, (n, length) in enumerate(bt.sizes):
        for i in range(n):
            p = length - n + i
            for mb, j, d, value in marks:
                if mb == b and j <= p and (not window or p - j < window or j < sinks):
                    kind[r, d] |= 1 if value == float("inf") else 2 if value == float("-inf") else 4
            r += 1
    kind = kind[:, None].expand(-1, bt.nq, -1)
    assert (out[kind == 1] == float("inf")).all() and (out[kind == 2] == float("-inf")).all()
    assert torch.isnan(out[kind >= 3]).all()
    rows = (kind == 0).reshape(bt.T, -1)
    check(out.reshape(bt.T, -1)[rows], (ref[0][rows], ref[1][rows]))


@pytest.mark.parametrize("table_extra", [0, 200])
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 4)])
@pytest.mark.parametrize("dh,nq,nkv", [(256, 8, 2), (128, 6, 2), (64, 3, 3)])
def test_prompt_values_that_are_not_finite(dh, nq, nkv, window, sinks, table_extra, dev):
    """Infinities and NaN in values that some rows of a chunk see and others do not: single dims and whole rows, at the
    start, inside and at the end of the sequences, opposite ones in one dim, keys split over blocks and not."""
    from qmtp import paged

    inf, nan = float("inf"), float("nan")
    bt = Batch([(150, 420), (70, 70), (5, 2), (33, 260)], nq, nkv, dh, 16, seed=dh + window, table_extra=table_extra)
    ref = attention_ref(bt, window, sinks)
    marks = [(0, 0, 3, inf), (0, 300, 7, -inf), (0, 330, 7, inf), (0, 419, 9, nan), (1, 2, 1, -inf), (2, 1, 4, inf),
             (3, 100, 11, inf), (3, 200, 12, nan), (3, 259, 13, -inf)]
    marks += [(1, 40, d, nan) for d in range(dh)]
    for b, j, d, value in marks:
        pg, sl = bt.rows(b, j)
        bt.v[pg, :, sl, d] = value
    bt.put(dev)
    call = lambda: paged.prompt_attention(*bt.args(), bt.d["cu"], gate=bt.d["gate"][:, :, 1], window=window, sinks=sinks)
    out = call()
    assert device_error() == 0
    check_classes(out, ref, bt, marks, window, sinks)
    assert torch.equal(call().view(torch.int16), out.view(torch.int16))


@pytest.mark.parametrize("dh,nq,nkv", [(256, 8, 2), (128, 8, 2), (64, 4, 4)])
def test_prompt_long_sequence_with_values_that_are_not_finite(dh, nq, nkv, dev):
    """16384 tokens with an infinite value early, and with a token late whose value is NaN: no wait runs out while rows are
    computed again, and what does not see them stays what it is without them."""
    from qmtp import paged

    T = 16384
    g = torch.Generator(device=dev).manual_seed(dh)
    rnd = lambda *s: torch.randn(s, generator=g, device=dev).to(BF16)
    cache = paged.PagedCache(rnd(T // 64, nkv, 64, dh), rnd(T // 64, nkv, 64, dh))
    q = rnd(T, nq, dh)
    table = torch.arange(T // 64, dtype=torch.int32, device=dev)[None]
    lens, cu = torch.tensor([T], dtype=torch.int32, device=dev), torch.tensor([0, T], dtype=torch.int32, device=dev)
    call = lambda c: paged.prompt_attention(q, c, table, lens, cu).view(T, nq, dh)
    clean = call(cache)
    # each of two results is this far from the exact one: its rounding, the weights', and the scores' error in the exponent
    # (|q . k| <= |q| |k|), against A = sum p |v|, which is itself a result within 2^-6 of the exact one
    A = call(paged.PagedCache(cache.k, cache.v.abs())).double() * (1 + 2.0 ** -6)
    e = dh ** -0.5 * dh * 2.0 ** -22 * float(q.float().norm(dim=-1).max() * cache.k.float().norm(dim=-1).max()) + 2.0 ** -20
    near = lambda a, rows: ((a[rows].double() - clean[rows].double()).abs()
                            <= 2 * (2.0 ** -8 * (1 + 2.0 ** -7) * clean[rows].double().abs() + (2.0 ** -8 + 2 * e) * A[rows])).all()
    held = cache.v.clone()
    cache.v[1, :, 36, 5] = float("inf")  # position 100
    out = call(cache)
    assert device_error() == 0
    assert (out[100:, :, 5] == float("inf")).all() and near(out, slice(0, 100))
    rest = torch.arange(dh, device=dev) != 5
    assert torch.equal(out[100:, :, rest], clean[100:, :, rest])
    cache.v.copy_(held)
    cache.v[16000 // 64, :, 0] = float("nan")
    out = call(cache)
    assert device_error() == 0
    assert torch.isnan(out[16000:]).all() and near(out, slice(0, 16000))
    assert torch.equal(out[:15800], clean[:15800])
    cache.v.fill_(float("nan"))
    assert torch.isnan(call(cache)).all() and device_error() == 0
