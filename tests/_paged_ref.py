"""64-bit reference of the paged-cache operators and the inputs of their tests."""
import torch

BF16 = torch.bfloat16
U = 2.0 ** -8  # half a bf16 step, relative


class Batch:
    """Sequences with (new, length) tokens over shuffled pages; tensors live on the CPU until put()."""

    def __init__(self, sizes, nq, nkv, dh, page, seed=0, spare=3, table_extra=0):
        g = torch.Generator().manual_seed(seed)
        self.sizes, self.nq, self.nkv, self.dh, self.page = sizes, nq, nkv, dh, page
        used = [-(-length // page) for _, length in sizes]
        self.pages = sum(used) + spare
        order = torch.randperm(self.pages, generator=g).to(torch.int32)
        self.table = torch.zeros((len(sizes), max(max(used), 1) + table_extra), dtype=torch.int32)
        at = 0
        for b, n in enumerate(used):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.lens = torch.tensor([length for _, length in sizes], dtype=torch.int32)
        self.cu = torch.tensor([0] + [n for n, _ in sizes]).cumsum(0).to(torch.int32)
        self.T = int(self.cu[-1])
        rnd = lambda *s: torch.randn(s, generator=g).to(BF16)
        self.k, self.v = rnd(self.pages, nkv, page, dh), rnd(self.pages, nkv, page, dh)
        self.q, self.gate = (rnd(self.T, nq, dh) * 1.5), rnd(self.T, nq, 2, dh)
        self.g = g

    def rows(self, b, pos):
        """(page, slot) of the positions pos of sequence b."""
        pos = torch.as_tensor(pos)
        return self.table[b].long()[pos // self.page], pos % self.page

    def put(self, dev):
        from qmtp.paged import PagedCache

        self.cache = PagedCache(self.k.to(dev), self.v.to(dev))
        self.d = {n: getattr(self, n).to(dev) for n in ("q", "gate", "table", "lens", "cu")}
        return self

    def args(self):
        return self.d["q"], self.cache, self.d["table"], self.d["lens"]


def visible(p, window, sinks):
    return [j for j in range(p + 1) if not window or p - j < window or j < sinks]


def attention_ref(bt: Batch, window=0, sinks=0, gate=True, scale=None):
    """(out, tol) float64 [T, nq * dh]: every row from its visible keys alone.

    tol is what fp32 sums and bf16 weights may be off: the output's rounding (U |out|), each weight's rounding
    (U times A = sum p |v|), and the scores' error e in the exponent (2 e A): dh products added in fp32, at
    most 2^-22 of sum |q k| each (the tensor core need not round to nearest), plus 2^-20 for exp and sums."""
    dh, G = bt.dh, bt.nq // bt.nkv
    scale = dh ** -0.5 if scale is None else scale
    out = torch.zeros((bt.T, bt.nq, dh), dtype=torch.float64)
    tol = torch.zeros_like(out)
    r = 0
    for b, (n, length) in enumerate(bt.sizes):
        for i in range(n):
            p = length - n + i
            keys = torch.tensor(visible(p, window, sinks), dtype=torch.long) if p >= 0 else torch.empty(0, dtype=torch.long)
            if len(keys):
                pg, sl = bt.rows(b, keys)
                for h in range(bt.nkv):
                    k, v = bt.k[pg, h, sl].double(), bt.v[pg, h, sl].double()
                    q = bt.q[r, h * G:(h + 1) * G].double()
                    p_ = torch.softmax(q @ k.T * scale, -1)
                    e = scale * dh * 2.0 ** -22 * (q.abs() @ k.abs().T).amax(-1, keepdim=True) + 2.0 ** -20
                    o, A = p_ @ v, p_ @ v.abs()
                    out[r, h * G:(h + 1) * G] = o
                    tol[r, h * G:(h + 1) * G] = U * o.abs() + (U + 2 * e) * A + 1e-30
            r += 1
    if gate:
        s = torch.sigmoid(bt.gate[:, :, 1].double())
        out, tol = out * s, tol * s * (1 + 2.0 ** -20)
    # a rounding of an already rounded value: second order
    return out.reshape(bt.T, -1), tol.reshape(bt.T, -1) * (1 + 2 * U)


def check(got, ref, rows=None):
    out, tol = ref
    got = got.double().cpu()
    if rows is not None:
        got, out, tol = got[rows], out[rows], tol[rows]
    bad = ~((got - out).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), float(((got - out).abs() / tol.clamp_min(1e-30)).nan_to_num(1e9).max()))


def append_ref(bt: Batch, qkv, gated, q_norm, k_norm, cos, sin, eps):
    """(q, q_tol, k, k_tol, v): k, v whole pools.  Each value is one bf16 rounding (U) off the 64-bit one, plus
    fp32 arithmetic: the mean of dh squares (dh 2^-24), root, divide and three products (8 2^-24), against
    the two products that a rotation adds."""
    T, dh, nq, nkv = bt.T, bt.dh, bt.nq, bt.nkv
    per = 2 if gated else 1
    x = qkv[:, : (nq * per + 2 * nkv) * dh].double().reshape(T, -1, dh)
    q, k, v = x[:, : nq * per: per], x[:, nq * per: nq * per + nkv], x[:, nq * per + nkv:]
    pos = torch.cat([torch.arange(length - n, length) for n, length in bt.sizes])

    def head(y, w):
        if w is not None:
            y = y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + eps) * w.double()
        mag = y.abs()
        if cos is not None:
            h = cos.shape[1]
            c, s = cos[pos.clamp_min(0)].double()[:, None], sin[pos.clamp_min(0)].double()[:, None]
            a, b = y[..., :h], y[..., h:2 * h]
            y = torch.cat([a * c - b * s, b * c + a * s, y[..., 2 * h:]], -1)
            mag = torch.cat([a.abs() * c.abs() + b.abs() * s.abs(), b.abs() * c.abs() + a.abs() * s.abs(), mag[..., 2 * h:]], -1)
        return y, U * y.abs() + (dh + 8) * 2.0 ** -24 * mag * (1 + U)

    q, q_tol = head(q, q_norm)
    kr, kr_tol = head(k, k_norm)
    kk, vv = bt.k.double(), bt.v.double()
    kt = torch.zeros_like(kk)
    r = 0
    for b, (n, length) in enumerate(bt.sizes):
        for i in range(n):
            p = length - n + i
            if p >= 0:
                pg, sl = bt.rows(b, p)
                kk[pg, :, sl], kt[pg, :, sl], vv[pg, :, sl] = kr[r + i], kr_tol[r + i], v[r + i]
        r += n
    return q, q_tol, kk, kt, vv
