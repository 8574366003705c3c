"""The serving operators' measured cases: attention over a paged key/value
cache (whole prompts, and single new tokens), the page operations of that
cache, and log probabilities of given tokens.

Each case has a plain form in elementary torch operations (`own` false) and the
calls a program makes of kernrt_b200 (`own` true); both work on the same inputs
and the same cache layout, [n_layers][2][n_pages][n_kv_heads][page_size][head_size]
with K at 0 and V at 1 of the second axis.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---- cases ------------------------------------------------------------------------


def listed():
    return [
        # a short prompt of a small model: one call's latency
        dict(name="prompt-128", op="attention", pages="bf16", heads=9, kv_heads=3, head=64, page=16, ctx="0", new="128"),
        # prompts of very different lengths packed into one step
        dict(name="prompt-ragged", op="attention", pages="bf16", heads=16, kv_heads=8, head=128, page=64,
             ctx="0,0,0,0,0,0", new="1,17,250,1023,2048,4095"),
        # one long prompt
        dict(name="prompt-8192", op="attention", pages="bf16", heads=24, kv_heads=8, head=64, page=32, ctx="0", new="8192"),
        # two prompts over an f32 cache, one kv head per head
        dict(name="prompt-f32", op="attention", pages="f32", heads=32, kv_heads=32, head=64, page=16, ctx="0,0", new="2048,1777"),
        # a prompt's later chunk behind a long context
        dict(name="chunk-512", op="attention", pages="bf16", heads=16, kv_heads=8, head=128, page=128, ctx="16001", new="512"),
        # one new token of one sequence: the latency of a decode step
        dict(name="decode-1", op="attention", pages="f32", heads=32, kv_heads=32, head=64, page=16, ctx="511", new="1"),
        # a serving batch: one new token of each of 64 sequences of ragged lengths
        dict(name="decode-64", op="attention", pages="bf16", heads=16, kv_heads=8, head=128, page=64,
             ctx=",".join(str(100 + (i * 2749) % 7900) for i in range(64)), new=",".join(["1"] * 64)),
        # one new token behind a very long context
        dict(name="decode-long", op="attention", pages="bf16", heads=24, kv_heads=8, head=64, page=32, ctx="131071", new="1"),
        # parallel samples of one prompt: 16 forks that each take a token of their own
        dict(name="fork-16", op="fork", pages="bf16", layers=24, kv_heads=32, head=64, page=32, length=1015, children=16),
        # a finished sequence leaves, the cache is compacted, the next one comes
        dict(name="compact", op="compact", pages="f32", layers=24, kv_heads=8, head=128, page=64, seqs=6, seq_pages=33),
        # the sampled token's log probability and the alternatives of one decode step
        dict(name="logprobs-1", op="logprobs", rows=1, vocab=151936, top=20, masked=0.0),
        # scoring a prompt
        dict(name="logprobs-1024", op="logprobs", rows=1024, vocab=49152, top=5, masked=0.0),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], evenly spread over its logarithm."""
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["prompt", "decode", "prompt", "decode", "fork", "compact", "logprobs", "logprobs"])
    pages = rng.choice(["bf16", "f32"])
    page = rng.choice([16, 32, 64, 128])
    if op in ("prompt", "decode"):
        head = rng.choice([64, 128, 64, 128, 8 * rng.randint(4, 16)])
        kv_heads = rng.randint(1, 16)
        heads = kv_heads * rng.choice([1, 2, 3, 4, 6, 8])
        if op == "prompt":
            # at most the largest listed prompt's scores, over a padded batch
            n = rng.choice([1, 1, 2, 3, 5, 8])
            most = int(math.sqrt(24 * 8192 * 8192 / (n * heads)))
            new = [_spread(rng, 1, min(8192, most)) for _ in range(n)]
            room = max(0, 24 * 8192 * 8192 // (n * heads * max(new)) - max(new))
            ctx = [rng.choice([0, 0, _spread(rng, 1, max(1, min(room, 20000)))]) if room > 1 else 0 for _ in range(n)]
        else:
            n = _spread(rng, 1, 128)
            most = max(16, min(131072, 3 * 10 ** 8 // (n * kv_heads * head)))
            top = _spread(rng, 16, most)
            ctx = [rng.randint(0, top) for _ in range(n)]
            new = [rng.choice([1, 1, 1, 2, 4]) for _ in range(n)] if rng.random() < 0.3 else [1] * n
        return dict(op="attention", pages=pages, heads=heads, kv_heads=kv_heads, head=head, page=page,
                    ctx=",".join(map(str, ctx)), new=",".join(map(str, new)))
    if op == "fork":
        kv_heads, head = rng.choice([1, 3, 8, 16, 32]), rng.choice([64, 128])
        return dict(op="fork", pages=pages, layers=rng.randint(1, 24), kv_heads=kv_heads, head=head, page=page,
                    length=_spread(rng, 1, 2000), children=_spread(rng, 1, 32 if kv_heads * page > 1024 else 64))
    if op == "compact":
        seqs = rng.randint(2, 8)
        kv_heads, head, layers = rng.choice([1, 3, 8, 16]), rng.choice([64, 128]), rng.randint(1, 24)
        per_page = layers * 2 * kv_heads * head * page * 4
        return dict(op="compact", pages=pages, layers=layers, kv_heads=kv_heads, head=head, page=page, seqs=seqs,
                    seq_pages=_spread(rng, 1, max(1, min(64, 2 * 10 ** 9 // (per_page * seqs)))))
    vocab = _spread(rng, 500, 200000)
    return dict(op="logprobs", rows=_spread(rng, 1, max(1, min(2048, 50 * 10 ** 6 // vocab))), vocab=vocab,
                top=rng.choice([0, 1, 5, 20, 32]), masked=rng.choice([0.0, 0.0, 0.5]))


def _ints(text):
    return [int(v) for v in text.split(",")]


def work(case):
    size = 2 if case.get("pages") == "bf16" else 4
    if case["op"] == "attention":
        ctx, new = _ints(case["ctx"]), _ints(case["new"])
        rows, row_kv = sum(new), case["kv_heads"] * case["head"]
        pairs = sum(n * c + n * (n + 1) // 2 for c, n in zip(ctx, new))  # (query, key) pairs that see each other
        return {"bytes": rows * 2 * case["heads"] * case["head"] * 4   # q read, out written
                + rows * 2 * row_kv * (4 + size)                       # new k and v read, stored
                + sum(ctx) * 2 * row_kv * size,                        # the context read
                "flops": 4 * case["head"] * case["heads"] * pairs}
    if case["op"] == "fork":
        rows = case["length"] % case["page"]  # the rows of the shared last page
        per = case["layers"] * 2 * case["kv_heads"] * case["head"] * size
        return {"bytes": max(1, (1 + case["children"]) * rows * per), "flops": 0}
    if case["op"] == "compact":
        per = case["layers"] * 2 * case["kv_heads"] * case["head"] * case["page"] * size
        return {"bytes": 2 * per * case["seq_pages"], "flops": 0}
    n = case["rows"] * case["vocab"]
    return {"bytes": 4 * n + case["rows"] * (12 + 8 * case["top"]), "flops": 4 * n}


# ---- inputs -----------------------------------------------------------------------


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _tables(case):
    """The page ids of each sequence: pages are taken lowest first while the
    sequences' contexts grow in four rounds, then for the new rows."""
    ctx, new, page = _ints(case["ctx"]), _ints(case["new"]), case["page"]
    rounds = [[c * r // 4 for c in ctx] for r in (1, 2, 3, 4)] + [[c + n for c, n in zip(ctx, new)]]
    tables, taken = [[] for _ in ctx], 0
    for lens in rounds:
        for t, n in zip(tables, lens):
            more = -(-n // page) - len(t)
            t.extend(range(taken, taken + more))
            taken += more
    return tables, taken


def _attention_inputs(case, seed):
    g = _gen(seed)
    rows = sum(_ints(case["new"]))
    tables, n_pages = _tables(case)
    qw, kw = case["heads"] * case["head"], case["kv_heads"] * case["head"]
    q = torch.randn(rows, qw, generator=g, device=DEV)
    k = torch.randn(rows, kw, generator=g, device=DEV)
    v = torch.randn(rows, kw, generator=g, device=DEV)
    kv = torch.empty(1, 2, n_pages, case["kv_heads"], case["page"], case["head"], dtype=DTYPES[case["pages"]], device=DEV)
    kv.normal_(generator=g)
    return q, k, v, kv, tables


def _logits(case, seed):
    g = _gen(seed)
    rows, vocab = case["rows"], case["vocab"]
    x = torch.randn(rows, vocab, generator=g, device=DEV) * 3
    targets = torch.randint(0, vocab, (rows,), generator=g, device=DEV, dtype=torch.int32)
    if case["masked"]:  # a constrained vocabulary: the masked tokens cannot be drawn
        out = torch.rand(rows, vocab, generator=g, device=DEV) < case["masked"]
        out.scatter_(1, targets[:, None].long(), False)
        x.masked_fill_(out, -math.inf)
    return x, targets


class _Holder:
    """Backend handles that go back to the backend with the state that made them."""

    def __init__(self, backend):
        self.backend, self.bufs, self.pages = backend, [], []

    def buf(self, rows):
        """A torch view of a new f32 (or int32) buffer, and its handle."""
        import kernrt_b200.interop as interop

        n = max(1, math.prod(rows))
        h = self.backend.alloc(n)
        self.backend.synchronize()  # its zeros are in place before torch's stream fills it
        self.bufs.append(h)
        return h, lambda dtype: self.kept(interop.as_torch(self.backend, h, rows, dtype))

    def kept(self, t):
        t.holder = self
        return t

    def filled(self, data):
        h, view = self.buf(tuple(data.shape))
        view(np.int32 if data.dtype == torch.int32 else np.float32).copy_(data)
        return h

    def cache(self, kind, n_layers, heads, kv_heads, head, page, n_pages, max_seqs, max_len):
        import kernrt_b200
        import kernrt_b200.interop as interop

        p = self.backend.pages_create(kernrt_b200.BF16 if kind == "bf16" else kernrt_b200.F32, n_layers, heads, kv_heads,
                                      head, page, n_pages, max_seqs, max_len)
        self.backend.synchronize()
        self.pages.append(p)
        view = interop.pages_as_torch(self.backend, p)
        return p, self.kept(view)

    def __del__(self):
        for p in self.pages:
            self.backend.pages_destroy(p)
        for h in self.bufs:
            self.backend.free(h)


_backends = []


def _backend():
    import kernrt_b200

    if not _backends:
        _backends.append(kernrt_b200.CudaBackend(0))
    return _backends[0]


def prepare(case, seed):
    state = dict(case=case)
    if case["op"] == "attention":
        q, k, v, kv, tables = _attention_inputs(case, seed)
        ctx, new = _ints(case["ctx"]), _ints(case["new"])
        if own:
            hold = state["hold"] = _Holder(_backend())
            b = hold.backend
            p, view = hold.cache(case["pages"], 1, case["heads"], case["kv_heads"], case["head"], case["page"],
                                 kv.shape[2], len(ctx), max(c + n for c, n in zip(ctx, new)))
            seqs = [b.seq_open(p) for _ in ctx]
            for r in (1, 2, 3, 4):
                b.pages_step(p, seqs, [c * r // 4 - c * (r - 1) // 4 for c in ctx])
            view.copy_(kv)
            b.pages_step(p, seqs, new)
            state.update(p=p, kv=view, q=hold.filled(q), k=hold.filled(k), v=hold.filled(v))
            state["out"], out = hold.buf(tuple(q.shape))
            state["out_view"] = out(np.float32)
            return state
        # what a program of the plain form keeps: padded tables, places of the new rows
        width = max(map(len, tables))
        tab = torch.tensor([t + [0] * (width - len(t)) for t in tables], device=DEV)
        seq = torch.tensor(np.repeat(np.arange(len(new)), new), device=DEV)
        at = torch.tensor(np.concatenate([np.arange(n) for n in new]), device=DEV)
        ctx_t = torch.tensor(ctx, device=DEV)
        state.update(q=q, k=k, v=v, kv=kv, tab=tab, seq=seq, at=at, ctx=ctx_t, most=max(new),
                     length=max(c + n for c, n in zip(ctx, new)))
        return state
    if case["op"] in ("fork", "compact"):
        g = _gen(seed)
        page = case["page"]
        if case["op"] == "fork":
            held = [-(-case["length"] // page)]
            lengths, n_pages = [case["length"]], held[0] + case["children"] * 2
        else:
            lengths = [case["seq_pages"] * page - 3] * case["seqs"]
            n_pages = case["seqs"] * case["seq_pages"] + case["seq_pages"]
        kv = torch.empty(case["layers"], 2, n_pages, case["kv_heads"], page, case["head"], dtype=DTYPES[case["pages"]],
                         device=DEV)
        kv.normal_(generator=g)
        if own:
            hold = state["hold"] = _Holder(_backend())
            b = hold.backend
            p, view = hold.cache(case["pages"], case["layers"], case["kv_heads"], case["kv_heads"], case["head"], page,
                                 n_pages, len(lengths) + case.get("children", 1), max(lengths) + 1)
            seqs = [b.seq_open(p) for _ in lengths]
            b.pages_step(p, seqs, lengths)
            view.copy_(kv)
            del kv
            state.update(p=p, kv=view, seqs=seqs)
            return state
        taken, tables = 0, []
        for n in lengths:
            tables.append(list(range(taken, taken + -(-n // page))))
            taken += len(tables[-1])
        state.update(kv=kv, tables=tables)
        return state
    x, targets = _logits(case, seed)
    rows = case["rows"]
    if own:
        hold = state["hold"] = _Holder(_backend())
        state.update(x=hold.filled(x), targets=hold.filled(targets))
        for name, shape, dtype in (("logprob", (rows,), np.float32), ("entropy", (rows,), np.float32),
                                   ("ids", (rows, case["top"]), np.int32), ("tops", (rows, case["top"]), np.float32)):
            if math.prod(shape):
                state[name], view = hold.buf(shape)
                state[name + "_view"] = view(dtype)
        return state
    state.update(x=x, targets=targets)
    return state


# ---- one pass ---------------------------------------------------------------------


def run(state):
    op = state["case"]["op"]
    if op == "attention":
        return _attention_own(state) if own else _attention_plain(state)
    if op == "fork":
        return _fork_own(state) if own else _fork_plain(state)
    if op == "compact":
        return _compact_own(state) if own else _compact_plain(state)
    return _logprobs_own(state) if own else _logprobs_plain(state)


def _attention_own(s):
    b = s["hold"].backend
    b.pages_write(s["p"], 0, s["k"], s["v"])
    b.pages_attention(s["p"], 0, s["q"], s["out"])
    return {"out": s["out_view"], "kv": s["kv"]}


def _attention_plain(s):
    c, kv = s["case"], s["kv"]
    h, hk, d, page = c["heads"], c["kv_heads"], c["head"], c["page"]
    rows, batch = s["q"].shape[0], s["tab"].shape[0]
    # the new rows into their places of the cache
    pos = s["ctx"][s["seq"]] + s["at"]
    ids, off = s["tab"][s["seq"], pos // page], pos % page
    kv[0, 0][ids, :, off] = s["k"].view(rows, hk, d).to(kv.dtype)
    kv[0, 1][ids, :, off] = s["v"].view(rows, hk, d).to(kv.dtype)
    # the sequences as one padded batch
    n_keys = s["length"]
    keys, vals = (kv[0, i][s["tab"]].permute(0, 2, 1, 3, 4).reshape(batch, hk, -1, d)[:, :, :n_keys].float() for i in (0, 1))
    q = torch.zeros(batch, s["most"], h, d, device=DEV)
    q[s["seq"], s["at"]] = s["q"].view(rows, h, d)
    q = q.view(batch, s["most"], hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(batch, hk, -1, d)
    x = torch.matmul(q, keys.transpose(2, 3)).view(batch, hk, h // hk, s["most"], n_keys) / math.sqrt(d)
    last = s["ctx"][:, None] + torch.arange(s["most"], device=DEV)
    hidden = torch.arange(n_keys, device=DEV) > last[..., None]
    x.masked_fill_(hidden[:, None, None], -math.inf)
    x -= x.amax(-1, keepdim=True)
    x.exp_()
    total = x.sum(-1, keepdim=True)
    beyond = torch.arange(n_keys, device=DEV) >= (s["ctx"] + torch.bincount(s["seq"], minlength=batch))[:, None]
    vals = vals.masked_fill(beyond[:, None, :, None], 0.0)
    o = torch.matmul(x.view(batch, hk, -1, n_keys), vals).view(batch, hk, h // hk, s["most"], d) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(batch, s["most"], h * d)
    return {"out": o[s["seq"], s["at"]], "kv": kv}


def _fork_own(s):
    c, b, p = s["case"], s["hold"].backend, s["p"]
    children = b.seq_fork(p, s["seqs"][0], c["length"], c["children"])
    b.pages_step(p, children, [1] * c["children"])
    tables = np.stack([b.seq_table(p, q) for q in children])
    b.seq_close(p, children)
    return {"kv": s["kv"], "tables": tables}


def _fork_plain(s):
    """Each child shares the parent's full pages and has the used rows of the
    last, partly filled one in a page of its own."""
    c, kv, parent = s["case"], s["kv"], s["tables"][0]
    used, full = c["length"] % c["page"], c["length"] // c["page"]
    own_pages = range(len(parent), len(parent) + c["children"])
    tables = np.array([parent[:full] + [p] for p in own_pages], dtype=np.int32)
    if used:
        kv[:, :, own_pages.start:own_pages.stop, :, :used] = kv[:, :, parent[full], None, :, :used]
    return {"kv": kv, "tables": tables}


def _compact_own(s):
    c, b, p = s["case"], s["hold"].backend, s["p"]
    b.seq_close(p, [s["seqs"].pop(0)])
    moved = b.pages_compact(p)
    s["seqs"].append(b.seq_open(p))
    b.pages_step(p, s["seqs"][-1:], [c["seq_pages"] * c["page"] - 3])
    return {"kv": s["kv"], "moved": moved, "tables": np.stack([b.seq_table(p, q) for q in s["seqs"]])}


def _compact_plain(s):
    """The highest pages in use move into the lowest free ones."""
    c, kv, tables = s["case"], s["kv"], s["tables"]
    tables.pop(0)
    used = set(sum(tables, []))
    dst = [p for p in range(len(used)) if p not in used]
    src = sorted((p for p in used if p >= len(used)), reverse=True)
    if src:
        kv[:, :, torch.tensor(dst, device=DEV)] = kv[:, :, torch.tensor(src, device=DEV)]
    new = dict(zip(src, dst))
    tables[:] = [[new.get(p, p) for p in t] for t in tables]
    tables.append(list(range(len(used), len(used) + c["seq_pages"])))
    return {"kv": kv, "moved": len(src), "tables": np.array(tables, dtype=np.int32)}


def _logprobs_own(s):
    c = s["case"]
    s["hold"].backend.logprobs(s["x"], c["rows"], c["vocab"], s["targets"], s["logprob"], s["entropy"], c["top"],
                               s.get("ids", 0), s.get("tops", 0))
    return {n: s[n + "_view"] for n in ("logprob", "entropy", "ids", "tops") if n in s}


def _logprobs_plain(s):
    x, top = s["x"], s["case"]["top"]
    shifted = x - x.amax(1, keepdim=True)
    e = shifted.exp()
    total = e.sum(1, keepdim=True)
    log_total = total.log()
    logp = shifted - log_total
    got = {"logprob": logp.gather(1, s["targets"][:, None].long())[:, 0],
           "entropy": -(torch.where(e > 0, logp, 0.0) * (e / total)).sum(1)}
    if top:
        order = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :top]
        got["ids"] = order.to(torch.int32)
        got["tops"] = logp.gather(1, order)
    return got


# ---- in 64 bits ---------------------------------------------------------------------


def exact(case, seed):
    if case["op"] == "attention":
        q, k, v, kv, tables = _attention_inputs(case, seed)
        hk, d, page = case["kv_heads"], case["head"], case["page"]
        group = case["heads"] // hk
        out, row = torch.empty(q.shape, dtype=torch.float64, device=DEV), 0
        for c, n, t in zip(_ints(case["ctx"]), _ints(case["new"]), tables):
            ids = torch.tensor(t, device=DEV)
            new_k, new_v = (x[row:row + n].to(kv.dtype).double().view(n, hk, d) for x in (k, v))
            for j in range(hk):
                past = [kv[0, i, ids, j].reshape(-1, d)[:c].double() for i in (0, 1)]
                keys = torch.cat((past[0], new_k[:, j]))
                vals = torch.cat((past[1], new_v[:, j]))
                for lo in range(0, n, 2048):
                    m = min(2048, n - lo)
                    mine = q[row + lo:row + lo + m].double().view(m, hk, group, d)[:, j]
                    dots = torch.einsum("mgd,ld->mgl", mine, keys) * d ** -0.5
                    see = torch.arange(c + n, device=DEV)[None] <= c + lo + torch.arange(m, device=DEV)[:, None]
                    p = torch.softmax(dots.where(see[:, None], dots.new_tensor(-math.inf)), -1)
                    o = torch.einsum("mgl,ld->mgd", p, vals)
                    out[row + lo:row + lo + m].view(m, hk, group, d)[:, j] = o
            row += n
        return {"out": out, "kv": None}
    if case["op"] == "logprobs":
        x, targets = _logits(case, seed)
        lse = torch.logsumexp(x.double(), 1, keepdim=True)
        logp = x.double() - lse
        got = {"logprob": logp[torch.arange(case["rows"], device=DEV), targets.long()],
               "entropy": -torch.special.xlogy(logp.exp(), logp.exp()).sum(1)}
        if case["top"]:
            got["ids"] = None
            got["tops"] = torch.topk(logp, case["top"], 1)[0]
        return got
    return None
