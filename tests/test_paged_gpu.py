"""Paged-cache operators (qmtp.paged) against 64-bit references: append and decode attention."""
import pytest
import torch

from tests._paged_ref import BF16, Batch, append_ref, attention_ref, check

pytestmark = pytest.mark.gpu


def no_error():
    from qmtp import _lib

    torch.cuda.synchronize()
    assert _lib.device_error() == 0


# ------------------------------------------------------------------------------------ append
def run_append(bt, dev, gated, norm, rotary, use_cu, ld_extra=0, seed=9, max_pos=None):
    from qmtp import paged

    g = torch.Generator().manual_seed(seed)
    width = (bt.nq * (2 if gated else 1) + 2 * bt.nkv) * bt.dh
    qkv = torch.randn((bt.T, width + ld_extra), generator=g).to(BF16)
    qn = (1 + 0.3 * torch.randn(bt.dh, generator=g)).to(BF16) if norm else None
    kn = (1 + 0.3 * torch.randn(bt.dh, generator=g)).to(BF16) if norm else None
    cos = sin = None
    if rotary:
        ang = torch.arange(max_pos or max(int(bt.lens.max()), 1))[:, None] * 1e4 ** (-torch.arange(rotary // 2) / (rotary // 2))
        cos, sin = ang.cos().float(), ang.sin().float()
    ref = append_ref(bt, qkv, gated, qn, kn, cos, sin, 1e-6)
    bt.put(dev)
    dd = lambda t: None if t is None else t.to(dev)
    qkv_d = dd(qkv)
    q, gate = paged.append_qkv(qkv_d, bt.cache, bt.d["table"], bt.d["lens"], bt.d["cu"] if use_cu else None,
                               n_heads=bt.nq, gated=gated, q_norm=dd(qn), k_norm=dd(kn), cos=dd(cos), sin=dd(sin))
    no_error()
    if gated:
        want = qkv[:, : 2 * bt.nq * bt.dh].reshape(bt.T, bt.nq, 2, bt.dh)[:, :, 1]
        assert torch.equal(gate.cpu(), want) and gate.data_ptr() == qkv_d.data_ptr() + 2 * bt.dh
    return q.cpu().double(), bt.cache.k.cpu().double(), bt.cache.v.cpu().double(), ref


@pytest.mark.parametrize("nq,nkv,dh,rotary,gated,page", [
    (16, 4, 256, 64, True, 64), (4, 2, 256, 256, False, 16), (32, 8, 128, 128, False, 16), (7, 1, 128, 48, True, 32),
    (12, 12, 64, 32, False, 128), (5, 5, 64, 64, True, 256), (3, 1, 64, 0, False, 16)])
@pytest.mark.parametrize("norm", [True, False])
def test_append_ragged(nq, nkv, dh, rotary, gated, page, norm, dev):
    bt = Batch([(1, 1), (5, 17), (0, 9), (33, 65), (2, 300)], nq, nkv, dh, page, seed=nq + dh)
    q, k, v, (rq, rqt, rk, rkt, rv) = run_append(bt, dev, gated, norm, rotary, True, ld_extra=8)
    assert ((q - rq).abs() <= rqt).all()
    assert ((k - rk).abs() <= rkt).all()  # untouched rows have tolerance 0
    assert torch.equal(v, rv)


@pytest.mark.parametrize("S", [1, 3])
def test_append_uniform_and_padding_slots(S, dev):
    """cu = None; a sequence shorter than S (an empty slot of a padded batch) writes only what exists."""
    bt = Batch([(S, 40), (S, 0), (S, 1), (S, 16)], 8, 2, 128, 16, seed=S)
    bt_q = torch.full((bt.T, 8, 128), 7.0, dtype=BF16, device=dev)
    from qmtp import paged

    qkv = torch.randn((bt.T, 12 * 128), generator=bt.g).to(BF16)
    ref = append_ref(bt, qkv, False, None, None, None, None, 0.0)
    bt.put(dev)
    paged.append_qkv(qkv.to(dev), bt.cache, bt.d["table"], bt.d["lens"], n_heads=8, out=bt_q)
    no_error()
    for b, (n, length) in enumerate(bt.sizes):
        for i in range(n):
            row = bt_q[b * S + i].cpu()
            want = qkv[b * S + i, : 8 * 128].reshape(8, 128) if length - n + i >= 0 else torch.full((8, 128), 7.0, dtype=BF16)
            assert torch.equal(row, want)
    assert torch.equal(bt.cache.k.cpu().double(), ref[2]) and torch.equal(bt.cache.v.cpu().double(), ref[4])


def test_append_leaves_rows_of_no_sequence(dev):
    from qmtp import paged

    bt = Batch([(4, 10), (3, 3)], 4, 2, 64, 16).put(dev)
    qkv = torch.randn((12, 8 * 64), device=dev).to(BF16)
    out = torch.full((12, 4, 64), 3.0, dtype=BF16, device=dev)
    cu = torch.tensor([2, 6, 9], dtype=torch.int32, device=dev)
    paged.append_qkv(qkv, bt.cache, bt.d["table"], bt.d["lens"], cu, n_heads=4, out=out)
    no_error()
    assert (out[:2] == 3).all() and (out[9:] == 3).all()
    assert torch.equal(out[2:9], qkv[2:9, :256].reshape(7, 4, 64))


def test_append_device_checks(dev):
    """Page numbers, lengths and positions that the arrays cannot hold write nothing and set the error word."""
    from qmtp import _lib, paged

    qkv = torch.randn((2, 4 * 64), device=dev).to(BF16)
    for change in ("page", "negative page", "length", "position"):
        bt = Batch([(1, 20), (1, 20)], 2, 1, 64, 16).put(dev)
        k0, v0 = bt.cache.k.clone(), bt.cache.v.clone()
        kw = {}
        if change == "page":
            bt.d["table"][0, 1] = bt.pages
        elif change == "negative page":
            bt.d["table"][0, 1] = -1
        elif change == "length":
            bt.d["lens"][0] = 33
        else:
            kw = dict(cos=torch.ones(19, 16, device=dev), sin=torch.zeros(19, 16, device=dev))
        paged.append_qkv(qkv, bt.cache, bt.d["table"], bt.d["lens"], n_heads=2, **kw)
        torch.cuda.synchronize()
        assert _lib.device_error() == 2, change
        pg, sl = bt.rows(1, 19)
        if change != "position":
            assert torch.equal(bt.cache.k[pg, 0, sl], qkv[1, 128:192]), change
            k0[pg, 0, sl], v0[pg, 0, sl] = qkv[1, 128:192], qkv[1, 192:]
        assert torch.equal(bt.cache.k, k0) and torch.equal(bt.cache.v, v0), change


# ------------------------------------------------------------------------------------ decode
LAYOUTS = [(16, 4, 256, 64), (4, 2, 256, 16), (32, 8, 128, 16), (7, 1, 128, 32), (12, 12, 64, 128), (40, 2, 64, 256),
           (64, 1, 128, 64)]


@pytest.mark.parametrize("nq,nkv,dh,page", LAYOUTS)
@pytest.mark.parametrize("S", [1, 3, 8])
def test_decode(nq, nkv, dh, page, S, dev):
    """Lengths from one token to several slabs, at and around tile, page and slab borders; an empty sequence and
    one with fewer tokens than S."""
    from qmtp import paged

    lengths = [S, S + 1, 0, 1, 15, 16, 63, 64, 65, 127, 128, 129, 300]
    bt = Batch([(S, n) for n in lengths], nq, nkv, dh, page, seed=S + dh).put(dev)
    out = paged.attention(*bt.args(), gate=bt.d["gate"][:, :, 1])
    no_error()
    check(out, attention_ref(bt))


@pytest.mark.parametrize("length", [1000, 4095, 4096, 4097, 4608, 9001])
@pytest.mark.parametrize("dh,S", [(256, 3), (128, 1), (64, 2)])
def test_decode_long(length, dh, S, dev):
    from qmtp import paged

    bt = Batch([(S, length), (S, 37)], 4, 2, dh, 64, seed=length).put(dev)
    out = paged.attention(*bt.args())
    no_error()
    check(out, attention_ref(bt, gate=False))


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 2), (64, 0), (100, 4), (128, 130), (1000, 4), (5000, 3),
                                          (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("S", [1, 4])
def test_decode_window(window, sinks, S, dev):
    from qmtp import paged

    bt = Batch([(S, n) for n in (1, 6, 64, 131, 700, 6000)], 6, 2, 128, 32, seed=window % 1000).put(dev)
    out = paged.attention(*bt.args(), gate=bt.d["gate"][:, :, 1], window=window, sinks=sinks, scale=0.2)
    no_error()
    check(out, attention_ref(bt, window, sinks, scale=0.2))


@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 3)])
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), torch.finfo(BF16).min])
def test_decode_masked_places_hold_anything(window, sinks, poison, dev):
    """Rows behind the end, pages of nobody, rows outside the window and the other new tokens' future rows may
    hold infinities or NaN; pages that no query needs may be given away (table entry -1)."""
    from qmtp import paged

    S = 3
    bt = Batch([(S, n) for n in (3, 20, 130, 333)], 8, 2, 128, 16, seed=3, table_extra=2)
    ref = attention_ref(bt, window, sinks)
    seen = torch.zeros(bt.pages, bt.page, dtype=torch.bool)
    need = torch.zeros_like(bt.table, dtype=torch.bool)
    for b, (n, length) in enumerate(bt.sizes):
        for p in range(length - n, length):
            if p >= 0:
                keys = torch.tensor(visible_list(p, window, sinks))
                pg, sl = bt.rows(b, keys)
                seen[pg, sl] = True
                need[b, keys // bt.page] = True
    for t in (bt.k, bt.v):
        t.transpose(1, 2)[~seen] = poison
    bt.table[~need] = -1
    bt.put(dev)
    out = paged.attention(*bt.args(), gate=bt.d["gate"][:, :, 1], window=window, sinks=sinks)
    no_error()
    check(out, ref)
    # the newest token's own row: the earlier new tokens do not see it
    pg, sl = bt.rows(3, 332)
    bt.cache.v[pg, :, sl] = poison
    bt.cache.k[pg, :, sl] = poison
    out = paged.attention(*bt.args(), gate=bt.d["gate"][:, :, 1], window=window, sinks=sinks)
    no_error()
    check(out, ref, rows=list(range(3 * S + 2)))


def visible_list(p, window, sinks):
    from tests._paged_ref import visible

    return visible(p, window, sinks)


def test_decode_infinite_value_that_is_seen(dev):
    """What a query sees does reach it: an infinite value gives an infinity, a NaN key a NaN row."""
    from qmtp import paged

    bt = Batch([(2, 200)], 2, 1, 64, 16).put(dev)
    pg, sl = bt.rows(0, 198)
    bt.cache.v[pg, 0, sl, 5] = float("inf")
    out = paged.attention(*bt.args()).view(2, 2, 64)
    no_error()
    assert (out[..., 5] == float("inf")).all() and torch.isfinite(out[..., :5]).all() and torch.isfinite(out[..., 6:]).all()
    pg, sl = bt.rows(0, 199)
    bt.cache.k[pg, 0, sl, 0] = float("nan")
    out = paged.attention(*bt.args()).view(2, 2, 64)
    no_error()
    assert torch.isnan(out[1]).all() and not torch.isnan(out[0]).any()


def test_decode_bits_do_not_depend_on_the_call(dev):
    """A token's row: the same bits alone, in a batch, as one of S new tokens, and with other pages."""
    from qmtp import paged

    bt = Batch([(3, 5000), (3, 77), (3, 1029)], 16, 4, 256, 64, seed=8).put(dev)
    full = paged.attention(*bt.args(), gate=bt.d["gate"][:, :, 1])
    win = paged.attention(*bt.args(), window=300, sinks=4)
    for b in range(3):
        for s in range(3):
            row = slice(3 * b + s, 3 * b + s + 1)
            lens = bt.d["lens"][b:b + 1] - 2 + s
            a = (bt.d["q"][row], bt.cache, bt.d["table"][b:b + 1], lens)
            assert torch.equal(paged.attention(*a, gate=bt.d["gate"][row, :, 1]), full[row])
            assert torch.equal(paged.attention(*a, window=300, sinks=4), win[row])
    # other page size
    k16 = torch.zeros((5000 // 16 + 1, 4, 16, 256), dtype=BF16, device=dev)
    v16 = torch.zeros_like(k16)
    pg, sl = bt.rows(0, torch.arange(5000))
    at = torch.arange(5000)
    k16[at // 16, :, at % 16] = bt.cache.k[pg, :, sl]
    v16[at // 16, :, at % 16] = bt.cache.v[pg, :, sl]
    t16 = torch.arange(k16.shape[0], dtype=torch.int32, device=dev)[None]
    got = paged.attention(bt.d["q"][:3], paged.PagedCache(k16, v16), t16, bt.d["lens"][:1], gate=bt.d["gate"][:3, :, 1])
    assert torch.equal(got, full[:3])
    no_error()


def test_decode_strides_and_streams(dev):
    """Row strides of q and the gate's head stride; a call on a side stream; a large batch of short sequences."""
    from qmtp import paged

    bt = Batch([(2, 100), (2, 260)], 4, 2, 64, 16, seed=4).put(dev)
    ref = attention_ref(bt)
    wide = torch.zeros((4, 4 * 64 + 24), dtype=BF16, device=dev)
    q = wide[:, :256].unflatten(1, (4, 64))
    q.copy_(bt.d["q"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = paged.attention(q, bt.cache, bt.d["table"], bt.d["lens"], gate=bt.d["gate"][:, :, 1])
    side.synchronize()
    check(out, ref)
    many = Batch([(1, 1 + i % 40) for i in range(700)], 2, 1, 64, 16, seed=5).put(dev)
    check(paged.attention(*many.args()), attention_ref(many, gate=False))
    no_error()


def test_decode_device_checks(dev):
    """A bad page reads as zeros, a bad length as an empty sequence; both set the error word."""
    from qmtp import _lib, paged

    bt = Batch([(1, 40), (1, 40)], 2, 1, 64, 16, seed=6).put(dev)
    good = paged.attention(*bt.args())
    no_error()
    for value in (bt.pages, -1, 2 ** 31 - 1):
        bt.d["table"][0, 1] = value
        out = paged.attention(*bt.args())
        torch.cuda.synchronize()
        assert _lib.device_error() == 2
        assert torch.isfinite(out).all() and torch.equal(out[1], good[1])
    for value in (49, -1, 2 ** 31 - 1):
        bt.d["lens"][0] = value
        out = paged.attention(*bt.args())
        torch.cuda.synchronize()
        assert _lib.device_error() == 2
        assert (out[0] == 0).all() and torch.equal(out[1], good[1])


def test_decode_in_a_graph_follows_the_device_state(dev):
    """One captured step (append + attention) replayed while the sequences grow, against eager calls."""
    from qmtp import paged

    bt = Batch([(1, 60), (1, 127), (1, 500)], 4, 2, 128, 16, seed=7, spare=8, table_extra=1)
    free = [p for p in range(bt.pages) if p not in set(bt.table.flatten().tolist())][:3]
    for b, (_, length) in enumerate(bt.sizes):
        bt.table[b, -(-length // 16)] = free[b]
    bt.put(dev)
    qkv = torch.randn((3, 8 * 128), device=dev).to(BF16)

    def step():
        q, _ = paged.append_qkv(qkv, bt.cache, bt.d["table"], bt.d["lens"], n_heads=4)
        return paged.attention(q, bt.cache, bt.d["table"], bt.d["lens"])

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(5):
        qkv.copy_(torch.randn((3, 8 * 128), device=dev))
        bt.d["lens"].add_(1)
        graph.replay()
        got = out.clone()
        assert torch.equal(got, step()), i
    no_error()


@pytest.mark.parametrize("nq,nkv,dh,S", [(16, 4, 256, 1), (16, 4, 256, 3), (8, 2, 128, 1), (14, 2, 128, 2), (16, 2, 128, 4),
                                         (4, 4, 64, 1), (8, 1, 64, 2), (8, 1, 64, 4)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (300, 4), (129, 200)])
def test_decode_one_launch_and_two_give_the_same_bits(nq, nkv, dh, S, window, sinks, dev):
    """Short tables run as one launch (the slabs of a row in a thread-block cluster), wide ones as two: a table row with
    spare entries at its end takes the other way over the same keys."""
    from qmtp import paged

    for length in (1, 128, 515, 1000, 2048):
        if length < S:
            continue
        bt = Batch([(S, length)], nq, nkv, dh, 64, seed=length + S).put(dev)
        q, cache, table, lens = bt.args()
        wide = torch.full((1, 1000), -1, dtype=torch.int32, device=dev)
        wide[:, : table.shape[1]] = table
        kw = dict(gate=bt.d["gate"][:, :, 1], window=window, sinks=sinks)
        one, two = paged.attention(q, cache, table, lens, **kw), paged.attention(q, cache, wide, lens, **kw)
        no_error()
        assert torch.equal(one, two), length
        check(one, attention_ref(bt, window, sinks))


def test_most_sequences(dev):
    """4096 sequences, the most a call takes: append, decode and prompt attention of one new token each."""
    from qmtp import paged

    bt = Batch([(1, 1 + i % 37) for i in range(4096)], 2, 1, 64, 16, seed=9).put(dev)
    ref = attention_ref(bt, gate=False)
    check(paged.attention(*bt.args()), ref)
    check(paged.prompt_attention(*bt.args(), bt.d["cu"]), ref)
    qkv = torch.randn((4096, 4 * 64), device=dev).to(BF16)
    q, _ = paged.append_qkv(qkv, bt.cache, bt.d["table"], bt.d["lens"], bt.d["cu"], n_heads=2)
    no_error()
    assert torch.equal(q, qkv[:, :128].reshape(4096, 2, 64))
    pg = bt.d["table"].long().gather(1, ((bt.d["lens"].long() - 1) // 16)[:, None])[:, 0]
    assert torch.equal(bt.cache.v[pg, 0, (bt.d["lens"].long() - 1) % 16], qkv[:, 192:])


def test_shared_pages(dev):
    """Two sequences that begin with the same pages (a shared prompt) and end on their own."""
    from qmtp import paged

    bt = Batch([(2, 100), (2, 90)], 4, 2, 128, 16, seed=10)
    bt.table[1, :4] = bt.table[0, :4]
    bt.put(dev)
    ref = attention_ref(bt)
    kw = dict(gate=bt.d["gate"][:, :, 1])
    check(paged.attention(*bt.args(), **kw), ref)
    check(paged.prompt_attention(*bt.args(), bt.d["cu"], **kw), ref)
    no_error()


def test_two_streams_at_once(dev):
    """Calls of one cache on two streams, each with its own workspace, many times."""
    from qmtp import paged

    bt = Batch([(3, 5000), (3, 3000)], 16, 4, 256, 64, seed=11).put(dev)
    other = bt.d["q"].flip(0).contiguous()
    want = [(paged.attention(q, *bt.args()[1:]), paged.prompt_attention(q, *bt.args()[1:], bt.d["cu"])) for q in (bt.d["q"], other)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, q in enumerate((bt.d["q"], other)):
            with torch.cuda.stream(streams[i]):
                got[i].append((paged.attention(q, *bt.args()[1:]), paged.prompt_attention(q, *bt.args()[1:], bt.d["cu"])))
    no_error()
    for i in range(2):
        assert all(torch.equal(a, want[i][0]) and torch.equal(b, want[i][1]) for a, b in got[i])


def test_broadcast_gate_and_huge_window(dev):
    """One gate row for all tokens (stride 0); a window beyond every position is no window's values."""
    from qmtp import paged

    bt = Batch([(2, 70)], 4, 2, 64, 16, seed=12)
    bt.gate[:] = bt.gate[:1]
    bt.put(dev)
    gate = bt.d["gate"][:1, :, 1].expand(2, 4, 64)
    for f in (paged.attention, lambda *a, **k: paged.prompt_attention(*a, bt.d["cu"], **k)):
        check(f(*bt.args(), gate=gate, window=2 ** 40, sinks=2 ** 33), attention_ref(bt))
    no_error()


def test_python_refuses_scales_beyond_fp32_and_missing_rows(dev):
    from qmtp import paged

    bt = Batch([(2, 70), (2, 40)], 4, 2, 64, 16, seed=13).put(dev)
    q, cache, table, lens = bt.args()
    for scale in (1e39, float("inf"), -0.1, 1e-60):
        with pytest.raises(ValueError):
            paged.attention(q, cache, table, lens, scale=scale)
        with pytest.raises(ValueError):
            paged.prompt_attention(q, cache, table, lens, bt.d["cu"], scale=scale)
    with pytest.raises(ValueError):
        paged.prompt_attention(q, cache, table, lens, None)
    with pytest.raises(ValueError):
        paged.attention(q, cache, table, lens[:, None])


def test_python_refusals(dev):
    from qmtp import paged

    bt = Batch([(2, 70), (2, 40)], 4, 2, 64, 16, seed=13).put(dev)
    q, cache, table, lens = bt.args()
    cu = bt.d["cu"]
    bad = [dict(q=q.float()), dict(q=q[:, :, :32]), dict(q=q[:, ::2]), dict(q=q[:1].expand(4, 4, 64)), dict(q=q[:3]),
           dict(table=table.long()), dict(table=table[:1]), dict(table=table[:, :0]), dict(lens=lens.long()), dict(lens=lens[:1]),
           dict(table=table.t().contiguous().t()), dict(window=-1), dict(sinks=-1), dict(scale=0.0), dict(scale=float("nan")),
           dict(gate=q[:2]), dict(gate=q.float()), dict(out=torch.empty(4, 256, device=dev)),
           dict(out=torch.empty(4, 512, device=dev, dtype=BF16)[:, :256])]
    for change in bad:
        kw = dict(q=q, table=table, lens=lens)
        kw.update(change)
        a = (kw.pop("q"), cache, kw.pop("table"), kw.pop("lens"))
        with pytest.raises(ValueError):
            paged.attention(*a, **kw)
        if "q" not in change or change["q"].shape[0] != 3:
            with pytest.raises(ValueError):
                paged.prompt_attention(*a, cu, **kw)
    with pytest.raises(NotImplementedError):
        paged.attention(q.repeat(5, 1, 1)[:18], cache, table, lens)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        paged.attention(q.cpu(), cache, table, lens)
    for c in (cu.long(), cu[:2]):
        with pytest.raises(ValueError):
            paged.prompt_attention(q, cache, table, lens, c)
    qkv = torch.zeros((4, 8 * 64), device=dev, dtype=BF16)
    w = torch.ones(64, device=dev, dtype=BF16)
    cos = torch.ones(80, 8, device=dev)
    for change in (dict(qkv=qkv[:, :500]), dict(qkv=qkv.float()), dict(qkv=qkv[:1].expand(4, 512)), dict(n_heads=0), dict(n_heads=5),
                   dict(gated=True), dict(q_norm=w[:32]), dict(k_norm=w.float()), dict(cos=cos), dict(cos=cos, sin=cos[:9]),
                   dict(cos=cos.double(), sin=cos.double()), dict(eps=-1.0), dict(cu=cu.long()), dict(qkv=qkv[:3])):
        kw = dict(qkv=qkv, n_heads=4)
        kw.update(change)
        with pytest.raises(ValueError):
            paged.append_qkv(kw.pop("qkv"), cache, table, lens, kw.pop("cu", None), **kw)
    with pytest.raises(NotImplementedError):
        paged.append_qkv(qkv, cache, table, lens, n_heads=4, cos=torch.ones(80, 12, device=dev), sin=torch.ones(80, 12, device=dev))
    empty = paged.append_qkv(qkv[:0], cache, table, lens, n_heads=4)[0]
    assert empty.shape == (0, 4, 64)
    assert paged.attention(q[:0], cache, table, lens).shape == paged.prompt_attention(q[:0], cache, table, lens, cu).shape == (0, 256)
    k = torch.zeros((4, 2, 16, 64), device=dev, dtype=BF16)
    for kk, vv in ((k, k[:3]), (k.float(), k.float()), (k[:, :, ::2], k[:, :, ::2]), (k[0], k[0])):
        with pytest.raises(ValueError):
            paged.PagedCache(kk, vv)
    no_error()


@pytest.mark.parametrize("T", [1, 200, 1000, 10000])
def test_append_many_rows(T, dev):
    """Each of the row counts at which the kernel deals its work differently: q, k and v against the formulas."""
    nq, nkv, dh, rot = 6, 2, 128, 64
    bt = Batch([(T // 3, T // 3 + 5), (T - T // 3, T - T // 3)], nq, nkv, dh, 64, seed=T)
    q, k, v, (rq, rqt, rk, rkt, rv) = run_append(bt, dev, True, True, rot, True)
    assert ((q - rq).abs() <= rqt).all()
    assert ((k - rk).abs() <= rkt).all()
    assert torch.equal(v, rv)
