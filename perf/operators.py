"""Measured cases of the paged-cache attention operators (qmtp.paged).

Three operators that serve several sequences from one pool of key/value pages, as a serving loop
runs them:

  append   per-head RMS norms of queries and keys, their position rotation, and the new keys and
           values written to their pages, one pass over the projection output (paged.append_qkv);
  decode   attention of the 1..8 newest tokens of every sequence over its pages (paged.attention);
  prompt   attention of a ragged batch of prompt chunks over the same pages (paged.prompt_attention);

the last two optionally with a sliding window and first tokens that stay visible, and with the
output gate of a gated attention layer.  A case gives the head layout, the page size and how many
new tokens and earlier tokens each sequence has; `own` selects the framework's kernels, otherwise
`run` is the plain form in elementary torch operations.
"""
import math
import os
import random
import sys

import torch

own = False

# the package's folder is not importable by name; the working folder is the repository's root
PACKAGE = os.path.join(os.getcwd(), "qwen-mtp-mac_b200")

BF16 = torch.bfloat16


# ---------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one verify step of a single conversation (two drafts behind the 512-token benchmark prompt)
        dict(name="append-verify", op="append", nq=16, nkv=4, dh=256, rot=64, gated=True, page=64, batch=1,
             new_lo=3, new_hi=3, old_lo=512, old_hi=512, sizes=1),
        # one decode step of a serving batch, ungated heads of 128 rotated whole, small pages
        dict(name="append-batch64", op="append", nq=32, nkv=8, dh=128, rot=128, gated=False, page=16, batch=64,
             new_lo=1, new_hi=1, old_lo=100, old_hi=1000, sizes=2),
        # long prompts of three sequences, one pass
        dict(name="append-prompt", op="append", nq=16, nkv=4, dh=256, rot=64, gated=True, page=64, batch=3,
             new_lo=2000, new_hi=7000, old_lo=0, old_hi=500, sizes=3),
        # plain decoding of one conversation: latency
        dict(name="decode-one", op="decode", nq=16, nkv=4, dh=256, gated=True, page=64, batch=1, new_lo=1, new_hi=1,
             old_lo=514, old_hi=514, window=0, sinks=0, sizes=4),
        # the verify step (last token and two drafts) at the end of the decoder's 2048-token context
        dict(name="decode-verify", op="decode", nq=16, nkv=4, dh=256, gated=True, page=64, batch=1, new_lo=3, new_hi=3,
             old_lo=2045, old_hi=2045, window=0, sinks=0, sizes=5),
        # one conversation over a very long document: the keys and values have to be split
        dict(name="decode-long", op="decode", nq=16, nkv=4, dh=256, gated=True, page=64, batch=1, new_lo=1, new_hi=1,
             old_lo=131070, old_hi=131070, window=0, sinks=0, sizes=6),
        # a ragged serving batch, heads of 128, small pages
        dict(name="decode-batch32", op="decode", nq=32, nkv=8, dh=128, gated=False, page=16, batch=32, new_lo=1,
             new_hi=1, old_lo=300, old_hi=16000, window=0, sinks=0, sizes=7),
        # verify steps of a batch whose layer looks back 1024 tokens and keeps the first 4
        dict(name="decode-window", op="decode", nq=16, nkv=4, dh=256, gated=True, page=32, batch=24, new_lo=3, new_hi=3,
             old_lo=700, old_hi=24000, window=1024, sinks=4, sizes=8),
        # the 512-token benchmark prompt: time to first token of one conversation
        dict(name="prompt-512", op="prompt", nq=16, nkv=4, dh=256, gated=True, page=64, batch=1, new_lo=512, new_hi=512,
             old_lo=0, old_hi=0, window=0, sinks=0, sizes=9),
        # a whole long prompt, causal
        dict(name="prompt-16k", op="prompt", nq=16, nkv=4, dh=256, gated=True, page=64, batch=1, new_lo=16384,
             new_hi=16384, old_lo=0, old_hi=0, window=0, sinks=0, sizes=10),
        # a long prompt through a layer with a sliding window and four first tokens that stay visible
        dict(name="prompt-window", op="prompt", nq=32, nkv=8, dh=128, gated=False, page=32, batch=1, new_lo=8000,
             new_hi=8000, old_lo=0, old_hi=0, window=1024, sinks=4, sizes=11),
        # chunks of several prompts behind contexts of odd lengths, seven query heads to a key head
        dict(name="prompt-chunks", op="prompt", nq=28, nkv=4, dh=128, gated=False, page=16, batch=5, new_lo=1,
             new_hi=1500, old_lo=0, old_hi=9000, window=0, sinks=0, sizes=12),
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    nq, nkv, dh, rot, gated = rng.choice([(16, 4, 256, 64, True), (8, 2, 256, 64, True), (32, 8, 128, 128, False),
                                          (28, 4, 128, 128, False), (20, 4, 128, 64, True), (64, 8, 64, 64, False),
                                          (12, 12, 64, 32, False), (8, 1, 256, 256, False)])
    case = dict(op=rng.choice(["append", "decode", "decode", "prompt", "prompt"]), nq=nq, nkv=nkv, dh=dh, gated=gated,
                page=rng.choice([16, 32, 64, 128]), sizes=rng.randrange(1 << 20))
    window, sinks = rng.choice([(0, 0), (0, 0), (_log(rng, 64, 4096), rng.choice([0, 1, 4, 7]))])
    if case["op"] == "append":
        tokens = _log(rng, 1, 12000)
        batch = min(tokens, _log(rng, 1, 64))
        n = tokens // batch
        old = _log(rng, 1, 1000)
        case.update(rot=rot, batch=batch, new_lo=max(1, n // 2), new_hi=n, old_lo=old // 3, old_hi=old)
    elif case["op"] == "decode":
        batch = _log(rng, 1, 64)
        n = rng.randint(1, 8)
        old = _log(rng, 1, 160000 // batch)
        case.update(batch=batch, new_lo=n, new_hi=n, old_lo=old // 4, old_hi=old, window=window, sinks=sinks)
    else:
        batch = _log(rng, 1, 12)
        n = max(1, _log(rng, 16, 12000) // batch)
        old = rng.choice([0, _log(rng, 1, 10000 // batch)])
        case.update(batch=batch, new_lo=max(1, n // 3), new_hi=n, old_lo=old // 2, old_hi=old, window=window,
                    sinks=sinks)
    return case


def _sizes(case):
    """(new tokens, tokens in the cache after this step) of every sequence; part of the case, not of the seed."""
    rng = random.Random(case["sizes"])
    out = []
    for _ in range(case["batch"]):
        n = rng.randint(case["new_lo"], case["new_hi"])
        out.append((n, n + rng.randint(case["old_lo"], case["old_hi"])))
    return out


def _visible(case, pos):
    """Keys that the query at position pos sees."""
    w = case.get("window", 0)
    if not w or pos + 1 <= w:
        return pos + 1
    return w + min(case["sinks"], pos + 1 - w)


def work(case):
    nq, nkv, dh = case["nq"], case["nkv"], case["dh"]
    sizes = _sizes(case)
    tokens = sum(n for n, _ in sizes)
    if case["op"] == "append":
        heads = nq + 2 * nkv
        return {"bytes": 2 * tokens * dh * heads * 2 + tokens * case["rot"] * 4, "flops": tokens * (nq + nkv) * dh * 8}
    keys = pairs = 0
    for n, length in sizes:
        pairs += sum(_visible(case, p) for p in range(length - n, length))
        w = case["window"]
        first = max(0, length - n - w + 1) if w else 0
        keys += length - first + min(case["sinks"] if w else 0, first)
    rows = 3 if case["gated"] else 2
    return {"bytes": keys * nkv * dh * 4 + rows * tokens * nq * dh * 2, "flops": 4 * pairs * nq * dh}


# ---------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    nq, nkv, dh, page = case["nq"], case["nkv"], case["dh"], case["page"]
    sizes = _sizes(case)
    tokens = sum(n for n, _ in sizes)
    width = max(-(-length // page) for _, length in sizes)
    used = sum(-(-length // page) for _, length in sizes)
    pages = used + 3

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device=dev, dtype=BF16).mul_(scale)

    # pages are handed out in no order, as after a while of serving
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    table = torch.zeros((len(sizes), width), dtype=torch.int32, device=dev)
    at = 0
    for b, (_, length) in enumerate(sizes):
        k = -(-length // page)
        table[b, :k] = order[at:at + k]
        at += k
    st = dict(case=case, sizes=sizes, table=table,
              lens=torch.tensor([length for _, length in sizes], dtype=torch.int32, device=dev),
              k=normal(pages, nkv, page, dh), v=normal(pages, nkv, page, dh))
    starts = [0]
    for n, _ in sizes:
        starts.append(starts[-1] + n)
    st["cu"] = torch.tensor(starts, dtype=torch.int32, device=dev)
    per = 2 if case["gated"] else 1
    if case["op"] == "append":
        st["qkv"] = normal(tokens, (nq * per + 2 * nkv) * dh)
        st["q_norm"] = (1.0 + 0.2 * torch.randn(dh, generator=g, device=dev)).to(BF16)
        st["k_norm"] = (1.0 + 0.2 * torch.randn(dh, generator=g, device=dev)).to(BF16)
        half = case["rot"] // 2
        inv = 1e7 ** (-torch.arange(half, dtype=torch.float64, device=dev) / half)
        ang = torch.arange(max(length for _, length in sizes), dtype=torch.float64, device=dev)[:, None] * inv
        st["cos"], st["sin"] = ang.cos().float(), ang.sin().float()
    else:
        # queries as append leaves them (RMS about 1) and the gate where the projection wrote it
        st["q"] = normal(tokens, nq, dh, scale=1.3)
        st["gate"] = normal(tokens, nq, 2, dh)[:, :, 1] if case["gated"] else None
    if own:
        if PACKAGE not in sys.path:
            sys.path.insert(0, PACKAGE)
        from qmtp import paged

        st["cache"] = paged.PagedCache(st["k"], st["v"])
    return st


# ---------------------------------------------------------------------------------------- one pass
def run(st):
    case = st["case"]
    if own:
        return _run_own(st, case)
    if case["op"] == "append":
        return _plain_append(st, case)
    return _plain_attention(st, case)


def _run_own(st, case):
    from qmtp import paged

    uniform = case["new_lo"] == case["new_hi"]
    if case["op"] == "append":
        q, _ = paged.append_qkv(st["qkv"], st["cache"], st["table"], st["lens"], None if uniform else st["cu"],
                                n_heads=case["nq"], gated=case["gated"], q_norm=st["q_norm"], k_norm=st["k_norm"],
                                cos=st["cos"], sin=st["sin"], eps=1e-6)
        return q, st["k"], st["v"]
    kw = dict(gate=st["gate"], window=case["window"], sinks=case["sinks"])
    if case["op"] == "decode":
        return paged.attention(st["q"], st["cache"], st["table"], st["lens"], **kw)
    return paged.prompt_attention(st["q"], st["cache"], st["table"], st["lens"], st["cu"], **kw)


def _plain_append(st, case):
    nq, nkv, dh, page, half = case["nq"], case["nkv"], case["dh"], case["page"], case["rot"] // 2
    qkv, cu = st["qkv"], st["cu"].long()
    tokens = qkv.shape[0]
    row = torch.arange(tokens, device=qkv.device)
    seq = (row[:, None] >= cu[None, 1:]).sum(1)
    pos = st["lens"].long()[seq] - cu[seq + 1] + row
    nqc = nq * dh * (2 if case["gated"] else 1)
    q = qkv[:, :nqc].reshape(tokens, nq, -1, dh)[:, :, 0].float()
    k = qkv[:, nqc:nqc + nkv * dh].reshape(tokens, nkv, dh).float()
    v = qkv[:, nqc + nkv * dh:].reshape(tokens, nkv, dh)
    c, s = st["cos"][pos][:, None], st["sin"][pos][:, None]

    def norm_rotate(x, w):
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.float()
        a, b = x[..., :half], x[..., half:2 * half]
        return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * half:]], -1).to(BF16)

    where, slot = st["table"][seq, pos // page].long(), pos % page
    st["k"][where, :, slot] = norm_rotate(k, st["k_norm"])
    st["v"][where, :, slot] = v
    return norm_rotate(q, st["q_norm"]), st["k"], st["v"]


def _plain_attention(st, case):
    nq, nkv, dh, page = case["nq"], case["nkv"], case["dh"], case["page"]
    q, w, sinks = st["q"], case["window"], case["sinks"]
    out = torch.empty((q.shape[0], nq * dh), dtype=BF16, device=q.device)
    r0 = 0
    for b, (n, length) in enumerate(st["sizes"]):
        where = st["table"][b, :-(-length // page)].long()
        k = st["k"][where].transpose(0, 1).reshape(nkv, -1, dh)[:, :length].float()
        v = st["v"][where].transpose(0, 1).reshape(nkv, -1, dh)[:, :length].float()
        key = torch.arange(length, device=q.device)
        for i in range(0, n, 1024):  # queries in blocks, which bounds the score matrix
            m = min(1024, n - i)
            rows = slice(r0 + i, r0 + i + m)
            pos = torch.arange(length - n + i, length - n + i + m, device=q.device)[:, None]
            seen = key <= pos
            if w:
                seen = seen & ((pos - key < w) | (key < sinks))
            x = q[rows].float().reshape(m, nkv, nq // nkv, dh).permute(1, 2, 0, 3).reshape(nkv, -1, dh)
            s = (x @ k.transpose(1, 2)).mul_(dh ** -0.5).reshape(nkv, -1, m, length)
            s = s.masked_fill_(~seen, float("-inf"))
            s = s.sub_(s.amax(-1, keepdim=True)).exp_()
            total = s.sum(-1, keepdim=True)
            o = (s.reshape(nkv, -1, length) @ v).reshape(nkv, -1, m, dh) / total
            o = o.permute(2, 0, 1, 3).reshape(m, nq, dh)
            if st["gate"] is not None:
                o = o / (1.0 + torch.exp(-st["gate"][rows].float()))
            out[rows] = o.reshape(m, nq * dh).to(BF16)
        r0 += n
    return out


# ---------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    f64 = torch.float64
    nq, nkv, dh, page = case["nq"], case["nkv"], case["dh"], case["page"]
    group = nq // nkv
    if case["op"] == "append":
        k, v = st["k"].to(f64), st["v"].to(f64)
        x = st["qkv"].to(f64)
        per = 2 if case["gated"] else 1
        q = torch.empty((x.shape[0], nq, dh), dtype=f64, device=x.device)
        half, r = case["rot"] // 2, 0

        def head(y, weight, cos, sin):  # y [n, dh], one head
            y = y / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / dh + 1e-6) * weight.to(f64)
            z = y.clone()
            z[:, :half] = y[:, :half] * cos - y[:, half:2 * half] * sin
            z[:, half:2 * half] = y[:, half:2 * half] * cos + y[:, :half] * sin
            return z

        for b, (n, length) in enumerate(st["sizes"]):
            at = torch.arange(length - n, length, device=x.device)
            cos, sin = st["cos"][at].to(f64), st["sin"][at].to(f64)
            pg, sl = st["table"][b].long()[at // page], at % page
            for h in range(nq):
                q[r:r + n, h] = head(x[r:r + n, h * per * dh:(h * per + 1) * dh], st["q_norm"], cos, sin)
            for h in range(nkv):
                c0 = (nq * per + h) * dh
                k[pg, h, sl] = head(x[r:r + n, c0:c0 + dh], st["k_norm"], cos, sin)
                v[pg, h, sl] = x[r:r + n, c0 + nkv * dh:c0 + nkv * dh + dh]
            r += n
        return q, k, v
    out = torch.zeros((st["q"].shape[0], nq, dh), dtype=f64, device=st["q"].device)
    r = 0
    for b, (n, length) in enumerate(st["sizes"]):
        at = torch.arange(length, device=out.device)
        pg, sl = st["table"][b].long()[at // page], at % page
        for h in range(nkv):
            kk, vv = st["k"][pg, h, sl].to(f64), st["v"][pg, h, sl].to(f64)
            for i in range(0, n, 512):
                m = min(512, n - i)
                p = torch.arange(length - n + i, length - n + i + m, device=out.device)
                hidden = at[None, :] > p[:, None]
                if case["window"]:
                    hidden |= (p[:, None] - at[None, :] >= case["window"]) & (at[None, :] >= case["sinks"])
                for hq in range(h * group, (h + 1) * group):
                    s = st["q"][r + i:r + i + m, hq].to(f64) @ kk.T / math.sqrt(dh)
                    s[hidden] = -math.inf
                    out[r + i:r + i + m, hq] = torch.exp(s - torch.logsumexp(s, -1, keepdim=True)) @ vv
        r += n
    if st["gate"] is not None:
        out *= torch.sigmoid(st["gate"].to(f64))
    return out.reshape(out.shape[0], nq * dh)
