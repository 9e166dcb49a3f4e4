"""The operators of a serving step over a paged key/value cache, as a program calls them, beside their plain form.

  append  new tokens of a batch of sequences: per-head norms of queries and keys, position rotation, store into pages
  attend  attention of those tokens over the pages
  copy    pages copied in every layer's key and value cache (a sequence that forks, a pool that is compacted)
  sample  a token per row of logits with temperature, top-k, top-p and min-p, from a given random number

A batch: sequence b has the rows row_start[b] .. row_start[b + 1] of the queries; they are the last of its context[b] rows in the
cache, whose pages stand in row b of the page table (entries behind the last page are -1).
"""
import math
import random

import numpy as np
import torch

own = False

F16 = {"fp16": torch.float16, "bf16": torch.bfloat16}
DEV = "cuda"


# ------------------------------------------------------------------ cases
def _attend(name, batch, new, context, heads, dtype="fp16", page=16, single=0.0, window=0, first=0, sink=False, lens=1):
    return {"name": name, "op": "attend", "batch": batch, "new_min": new[0], "new_max": new[1], "ctx_min": context[0],
            "ctx_max": context[1], "hq": heads[0], "hkv": heads[1], "hd": heads[2], "dtype": dtype, "page": page, "single": single,
            "window": window, "first": first, "sink": sink, "lens": lens}


def _append(name, batch, new, context, heads, dtype="fp16", page=16, single=0.0, norm=True, lens=1):
    c = _attend(name, batch, new, context, heads, dtype, page, single, lens=lens)
    c.update(op="append", norm=norm)
    return c


def listed():
    return [
        # one stream, short context: the call's latency
        _attend("attend 1 token", 1, (1, 1), (500, 500), (32, 8, 128)),
        # a server's decode step: 64 streams of all ages
        _attend("attend 64 streams", 64, (1, 1), (150, 8192), (32, 8, 128), lens=2),
        # eight streams with narrow heads, a sliding window whose first tokens stay visible, sink logits
        _attend("attend 8 windowed", 8, (1, 1), (4000, 4200), (64, 8, 64), "bf16", 32, window=1024, first=4, sink=True, lens=3),
        # the prompt of one stream
        _attend("attend prompt 512", 1, (512, 512), (512, 512), (32, 8, 128)),
        # long prompts in chunks, far into their contexts
        _attend("attend chunks 2048", 2, (1900, 2048), (12000, 16384), (32, 8, 128), "bf16", 64, lens=4),
        # decode steps and chunks of prompts in one batch, odd lengths
        _attend("attend mixed", 24, (33, 700), (200, 6001), (32, 4, 128), "fp16", 32, single=0.7, lens=5),
        # a decode step's tokens into the cache
        _append("append 64 tokens", 64, (1, 1), (150, 8192), (32, 8, 128), lens=6),
        # a prompt's chunks into the cache
        _append("append chunks", 3, (900, 1600), (1600, 9001), (32, 8, 128), "bf16", 32, lens=7),
        # one sequence forks inside a page: its last page, in all layers
        {"name": "copy fork", "op": "copy", "layers": 36, "pages": 64, "page": 16, "hkv": 8, "hd": 128, "pairs": 3, "dtype": "fp16"},
        # a pool is compacted
        {"name": "copy compact", "op": "copy", "layers": 24, "pages": 300, "page": 64, "hkv": 8, "hd": 64, "pairs": 133, "dtype": "bf16"},
        # one stream's next token
        {"name": "sample 1 row", "op": "sample", "rows": 1, "vocab": 151936, "temperature": 0.6, "top_k": 20, "top_p": 0.95, "min_p": 0.0},
        # a server's next tokens
        {"name": "sample 128 rows", "op": "sample", "rows": 128, "vocab": 201088, "temperature": 1.0, "top_k": 0, "top_p": 0.9, "min_p": 0.02},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


HEADS = [(32, 8, 128), (32, 4, 128), (64, 8, 64), (12, 12, 64), (24, 8, 96), (8, 1, 128), (14, 2, 64), (40, 8, 128)]


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "copy", "sample"])
    dtype, page = rng.choice(["fp16", "bf16"]), rng.choice([16, 32, 64, 128, 256])
    heads, lens = rng.choice(HEADS), rng.randrange(1, 1 << 20)
    if op == "attend":
        window, first = (rng.choice([100, 512, 1024, 4096]), rng.choice([0, 1, 4, 64])) if rng.random() < 0.3 else (0, 0)
        sink = rng.random() < 0.25
        if rng.random() < 0.5:  # tokens one by one, or a few (drafts) at a time
            batch, new = _log(rng, 1, 96), (1, rng.choice([1, 1, 1, 2, 4, 9]))
            hi = _log(rng, 64, min(32768, 500000 // batch))
            single = 0.0
        else:  # chunks, alone or among single tokens
            batch = _log(rng, 1, 24)
            hi = _log(rng, 64, min(16384, 120000 // batch))
            most = max(2, min(2048, hi, int(3.0e8 / (batch * hi))))
            n = _log(rng, 2, most)
            new, single = (max(1, n // 2), n), rng.choice([0.0, 0.0, 0.6])
        return _without_name(_attend("", batch, new, (max(1, hi // rng.choice([1, 2, 8])), hi), heads, dtype, page, single, window, first, sink, lens))
    if op == "append":
        batch = _log(rng, 1, 128)
        n = _log(rng, 1, max(1, 4096 // batch))
        hi = max(n, _log(rng, 64, 16384))
        return _without_name(_append("", batch, (max(1, n // 2), n), (max(1, hi // 4), hi), heads, dtype, page, rng.choice([0.0, 0.5]), rng.random() < 0.8, lens))
    if op == "copy":
        hkv, hd, layers = heads[1], heads[2], rng.choice([1, 4, 24, 36, 48])
        room = int(1.6e9 / (layers * 4 * page * hkv * hd))  # pages of a pool of 1.6 GB
        pages = max(4, min(room, _log(rng, 8, 400)))
        return {"op": "copy", "layers": layers, "pages": pages, "page": page, "hkv": hkv, "hd": hd, "pairs": _log(rng, 1, max(1, pages // 2 - 1)), "dtype": dtype}
    return {"op": "sample", "rows": _log(rng, 1, 128), "vocab": rng.choice([32000, 50257, 128256, 151936, 201088]), "temperature": round(rng.uniform(0.4, 1.3), 3),
            "top_k": rng.choice([0, 0, 1, _log(rng, 2, 1000)]), "top_p": rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]),
            "min_p": rng.choice([0.0, 0.0, round(rng.uniform(0.005, 0.2), 4)])}


def _without_name(c):
    return {k: v for k, v in c.items() if k != "name"}


def _lengths(c):
    """New tokens and context of every sequence: they belong to the case."""
    r = random.Random(c["lens"])
    new, ctx = [], []
    for b in range(c["batch"]):
        n = 1 if r.random() < c["single"] and b else r.randint(c["new_min"], c["new_max"])
        new.append(n)
        ctx.append(max(n, r.randint(c["ctx_min"], c["ctx_max"])))
    new[0], ctx[0] = c["new_max"], max(c["new_max"], c["ctx_max"])
    return new, ctx


# ------------------------------------------------------------------ inputs
def _batch(c, r, g):
    new, ctx = _lengths(c)
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    ps = c["page"]
    need = [-(-n // ps) for n in ctx]
    pool = sum(need) + 3
    ids = torch.randperm(pool, generator=g).to(torch.int32)
    table, at = torch.full((len(new), max(need)), -1, dtype=torch.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    return {"table": table.to(DEV), "row_start": i32(start), "context": i32(ctx), "max_new": max(new), "max_rows": max(ctx), "tokens": start[-1], "pool": pool}


def prepare(case, seed):
    g, cpu = torch.Generator(device=DEV).manual_seed(seed), torch.Generator().manual_seed(seed)
    rnd = lambda shape, dtype=torch.float32: torch.randn(shape, generator=g, device=DEV, dtype=dtype)  # noqa: E731
    s = dict(case)
    if case["op"] in ("attend", "append"):
        s.update(_batch(case, None, cpu))
        t, hq, hkv, hd = F16[case["dtype"]], case["hq"], case["hkv"], case["hd"]
        shape = (s["pool"], case["page"], hkv, hd)
        if case["op"] == "attend":
            # scores of a few units: some rows of the cache stand out, as in a trained model
            s.update(q=(2 * rnd((s["tokens"], hq, hd))).to(t), k=rnd(shape, t), v=rnd(shape, t), sinks=rnd((hq,)) if case["sink"] else None)
        else:
            # one projection's rows hold q | k | v
            qkv = rnd((s["tokens"], (hq + 2 * hkv) * hd))
            angle = torch.arange(s["max_rows"], dtype=torch.float64)[:, None] * 1e6 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)[None]
            angle = torch.cat([angle, angle], 1)
            s.update(q=qkv[:, :hq * hd], knew=qkv[:, hq * hd:(hq + hkv) * hd], vnew=qkv[:, (hq + hkv) * hd:], k=rnd(shape, t), v=rnd(shape, t),
                     cos=angle.cos().float().to(DEV), sin=angle.sin().float().to(DEV), eps=1e-6,
                     gq=1 + 0.1 * rnd((hd,)) if case["norm"] else None, gk=1 + 0.1 * rnd((hd,)) if case["norm"] else None)
    elif case["op"] == "copy":
        s["kv"] = rnd((case["layers"], 2, case["pages"], case["page"], case["hkv"], case["hd"]), F16[case["dtype"]])
        ids, n = torch.randperm(case["pages"], generator=cpu).to(torch.int32), case["pairs"]
        s["dst"], s["src"] = ids[:n].to(DEV), ids[n:][torch.randint(case["pages"] - n, (n,), generator=cpu)].to(DEV)
    else:
        # a broad bulk and some tokens that stand out
        x = 2 * rnd((case["rows"], case["vocab"]))
        at = torch.randint(case["vocab"], (case["rows"], 48), generator=g, device=DEV)
        x.scatter_add_(1, at, 7 + 3 * rnd((case["rows"], 48)))
        s.update(logits=x, u=torch.rand(case["rows"], generator=g, device=DEV))
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    if own:
        return _run_own(s)
    return {"attend": _plain_attend, "append": _plain_append, "copy": _plain_copy, "sample": _plain_sample}[s["op"]](s)


def _run_own(s):
    from nntrainer_b200 import backend as be
    if s["op"] == "attend":
        return be.paged_attention(s["q"], s["k"], s["v"], s["table"], s["row_start"], s["context"], s["max_new"], s["max_rows"],
                                  window=s["window"] or None, first_tokens=s["first"], sink=s["sinks"])
    if s["op"] == "append":
        q = be.paged_append(s["q"], s["knew"], s["vnew"], s["k"], s["v"], s["table"], s["row_start"], s["context"], s["max_new"],
                            s["cos"], s["sin"], qk_norm=(s["gq"], s["gk"], s["eps"]) if s["norm"] else None)
        return {"q": q, "k": s["k"], "v": s["v"]}
    if s["op"] == "copy":
        be.copy_pages(s["kv"], s["src"], s["dst"])
        return s["kv"]
    idx, _, prob = be.sample(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
    return {"id": idx, "prob": prob}


def _seq_of(s):
    """Sequence of every query row, its place among the sequence's new tokens, and its position."""
    tok = torch.arange(s["tokens"], device=DEV)
    seq = torch.searchsorted(s["row_start"].long(), tok, right=True) - 1
    at = tok - s["row_start"][seq]
    new = (s["row_start"][1:] - s["row_start"][:-1])[seq]
    return seq, at, s["context"][seq] - new + at


def _plain_attend(s):
    start, ctx, T, L, hq, hkv, hd, ps = s["row_start"], s["context"], s["max_new"], s["max_rows"], s["hq"], s["hkv"], s["hd"], s["page"]
    B, G, t = ctx.numel(), s["hq"] // s["hkv"], s["q"].dtype
    i, j = torch.arange(T, device=DEV), torch.arange(L, device=DEV)
    new = start[1:] - start[:-1]
    Q = s["q"][(start[:-1, None] + i).clamp(max=s["tokens"] - 1)].float()  # [B, T, hq, hd]
    Q = Q.view(B, T, hkv, G, hd).permute(0, 2, 3, 1, 4).reshape(B, hkv, G * T, hd)
    page = s["table"][:, j // ps].clamp(min=0).long()
    K, V = (x[page, j % ps].float().permute(0, 2, 1, 3) for x in (s["k"], s["v"]))  # [B, hkv, L, hd]
    pos = (ctx - new)[:, None] + i
    seen = j <= pos[..., None]
    if s["window"]:
        seen &= (j > pos[..., None] - s["window"]) | (j < s["first"])
    S = (Q @ K.transpose(2, 3)).mul_(1 / math.sqrt(hd)).view(B, hkv, G, T, L).masked_fill_(~seen[:, None, None], -math.inf)
    m = S.amax(-1, keepdim=True)
    sink = s["sinks"].view(1, hkv, G, 1, 1) if s["sink"] else None
    if sink is not None:
        m = torch.maximum(m, sink)
    m = m.masked_fill(m == -math.inf, 0.0)
    S.sub_(m).exp_()
    total = S.sum(-1, keepdim=True)
    if sink is not None:
        total = total + (sink - m).exp()
    O = (S.view(B, hkv, G * T, L) @ V).view(B, hkv, G, T, hd) / total.masked_fill(total == 0, 1.0)
    O = O.permute(0, 3, 1, 2, 4).reshape(B * T, hq, hd)
    seq, at, _ = _seq_of(s)
    return O[seq * T + at].to(t)


def _plain_append(s):
    hq, hkv, hd, t = s["hq"], s["hkv"], s["hd"], s["k"].dtype
    seq, _, pos = _seq_of(s)

    def turned(x, heads, gamma):
        x = x.reshape(-1, heads, hd).float()
        if gamma is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"]) * gamma
        c, n = s["cos"][pos][:, None, :hd // 2], s["sin"][pos][:, None, :hd // 2]
        a, b = x[..., :hd // 2], x[..., hd // 2:]
        return torch.cat([a * c - b * n, a * n + b * c], -1).to(t)

    page = s["table"][seq, pos // s["page"]].long()
    s["k"][page, pos % s["page"]] = turned(s["knew"], hkv, s["gk"])
    s["v"][page, pos % s["page"]] = s["vnew"].reshape(-1, hkv, hd).to(t)
    return {"q": turned(s["q"], hq, s["gq"]), "k": s["k"], "v": s["v"]}


def _plain_copy(s):
    s["kv"][:, :, s["dst"].long()] = s["kv"][:, :, s["src"].long()]
    return s["kv"]


def _plain_sample(s):
    # in 64 bits: a cumulative sum is compared with a number that falls anywhere between two of its values
    x, n = s["logits"], s["vocab"]
    w = ((x.double() - x.amax(-1, keepdim=True).double()) / s["temperature"]).exp_()
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    cum = ws.cumsum(-1)
    k = s["top_k"] if 0 < s["top_k"] < n else n
    keep = (torch.arange(n, device=DEV) < k) & (ws >= s["min_p"])
    if s["top_p"] < 1:
        keep &= cum - ws < s["top_p"] * cum[:, k - 1:k]
    keep[:, 0] = True
    w = w * torch.zeros_like(keep).scatter_(1, order, keep)
    cum = w.cumsum(-1)
    idx = (cum <= s["u"].double()[:, None] * cum[:, -1:]).sum(-1, keepdim=True).clamp(max=n - 1)
    return {"id": idx[:, 0].int(), "prob": (w.gather(1, idx)[:, 0] / cum[:, -1]).float()}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["op"] in ("attend", "append"):
        new, ctx = _lengths(case)
        hq, hkv, hd = case["hq"], case["hkv"], case["hd"]
        if case["op"] == "append":
            elements = sum(new) * (hq + 2 * hkv) * hd
            return {"bytes": 6 * elements + 4 * hd * len({c - i for n, c in zip(new, ctx) for i in range(n)}), "flops": 8 * elements}
        pairs = rows = 0
        for n, c in zip(new, ctx):
            w, f = case["window"] or c, case["first"]
            # rows seen by the query at position p: the window's, and the first ones in front of it
            pairs += sum(min(p + 1, w) + min(f, max(0, p + 1 - w)) for p in range(c - n, c))
            rows += min(c, w + n - 1) + min(f, max(0, c - n + 1 - w))
        return {"bytes": 4 * rows * hkv * hd + 4 * sum(new) * hq * hd, "flops": 4 * pairs * hq * hd}
    if case["op"] == "copy":
        return {"bytes": 4 * 2 * case["layers"] * case["pairs"] * case["page"] * case["hkv"] * case["hd"], "flops": 0}
    return {"bytes": 4 * case["rows"] * case["vocab"], "flops": 4 * case["rows"] * case["vocab"]}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "copy":  # nothing is computed: the values themselves
        kv, src, dst = s["kv"], s["src"].tolist(), s["dst"].tolist()
        moved = {d: kv[:, :, a].clone() for a, d in zip(src, dst)}
        for d, page in moved.items():
            kv[:, :, d] = page
        return kv
    if case["op"] == "sample":
        prob, u = np.empty(case["rows"]), s["u"].double().cpu().numpy()
        for r, x in enumerate(s["logits"].double().cpu().numpy()):
            order = np.argsort(-x, kind="stable")
            if 0 < case["top_k"] < x.size:
                order = order[:case["top_k"]]
            p = np.exp((x[order] - x[order[0]]) / case["temperature"])
            m = 1 + int(np.searchsorted(np.cumsum(p), case["top_p"] * p.sum())) if case["top_p"] < 1 else p.size
            m = max(1, min(m, int(np.count_nonzero(p >= case["min_p"]))))
            kept = np.sort(order[:m])
            p = np.exp((x[kept] - x[order[0]]) / case["temperature"])
            c = np.cumsum(p)
            prob[r] = p[min(int(np.searchsorted(c, u[r] * c[-1], side="right")), m - 1)] / c[-1]
        return {"id": None, "prob": torch.from_numpy(prob)}
    new, ctx = _lengths(case)
    hq, hkv, hd, ps = case["hq"], case["hkv"], case["hd"], case["page"]
    G, table = hq // hkv, s["table"].long()
    if case["op"] == "append":
        q, k, v, at = [], s["k"].double(), s["v"].double(), 0
        cos, sin = s["cos"].double(), s["sin"].double()

        def turned(x, heads, gamma, pos):
            z = torch.view_as_complex(torch.stack(_halves(x.double().reshape(-1, heads, hd), gamma, s["eps"]), -1))
            z = z * torch.complex(cos[pos, :hd // 2], sin[pos, :hd // 2])[:, None]
            return torch.cat([z.real, z.imag], -1)

        for b, (n, c) in enumerate(zip(new, ctx)):
            pos = torch.arange(c - n, c, device=DEV)
            page = table[b][torch.div(pos, ps, rounding_mode="floor")]
            q.append(turned(s["q"][at:at + n], hq, s["gq"], pos))
            k[page, pos % ps] = turned(s["knew"][at:at + n], hkv, s["gk"], pos)
            v[page, pos % ps] = s["vnew"][at:at + n].double().reshape(n, hkv, hd)
            at += n
        return {"q": torch.cat(q), "k": k, "v": v}
    out, at = [], 0
    for b, (n, c) in enumerate(zip(new, ctx)):
        pages = table[b, :-(-c // ps)]
        K, V = (x[pages].reshape(-1, hkv, hd)[:c].double() for x in (s["k"], s["v"]))
        Q = s["q"][at:at + n].double()
        at += n
        p, j = torch.arange(c - n, c, device=DEV)[:, None], torch.arange(c, device=DEV)[None]
        hidden = j > p
        if case["window"]:
            hidden = hidden | ((j <= p - case["window"]) & (j >= case["first"]))
        heads = []
        for h in range(hq):
            score = (Q[:, h] @ K[:, h // G].T) / math.sqrt(hd)
            score[hidden] = -math.inf
            if case["sink"]:
                score = torch.cat([score, s["sinks"][h].double().expand(n, 1)], 1)
            weight = torch.softmax(score, 1)[:, :c]
            heads.append(weight @ V[:, h // G])
        out.append(torch.stack(heads, 1))
    return torch.cat(out)


def _halves(x, gamma, eps):
    if gamma is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * gamma.double()
    return x[..., :x.shape[-1] // 2], x[..., x.shape[-1] // 2:]
