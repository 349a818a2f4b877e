"""What the speed of decoding several sequences over a paged cache is measured on.

A step of several conversations, or of several continuations of one prompt: the new rows into the pages
of an f16 cache (sg_gpu_run_page_store), attention of each sequence's one new token over its pages, which
also sums the weight that every cached row was given (sg_gpu_run_attn_paged), the eviction of the rows
that were given least (sg_gpu_run_page_evict), and the next tokens, sampled from given random numbers
(sg_gpu_run_sample). Head layouts, head_dim and vocabulary are this repository's model configurations or
generic.

The cache: K and V pools f16 [pages][page][kv head][hd], a table int32 [sequence][width] of page numbers;
slot j of a sequence lies in page table[j / page] at row j % page. Beside it, per sequence, kv head and
slot: the weight f32 and the position int32 of the row that the slot holds.

Where `own` is false every operator is computed from elementary torch operations.
"""
import ctypes as C
import math

import numpy as np
import torch

own = False

KINDS = ("store", "attn", "evict", "sample")
VOCAB = 151936

# (query heads, kv heads, head dim): this engine's two models and its micro configuration, then generic ones.
HEADS = ((24, 4, 256), (8, 2, 256), (16, 4, 256), (32, 8, 128), (12, 12, 64), (16, 1, 128))
ELEMENTS = 262000 * 4 * 256         # of K in the largest attention


def listed():
    return [
        # The new tokens of a batch of conversations, one row each: latency.
        {"name": "store_step", "kind": "store", "seqs": 16, "rows": 1, "kv_heads": 4, "head_dim": 256, "page": 16, "slot": 3000},
        # A prompt behind a first turn that ends inside a page.
        {"name": "store_prompt", "kind": "store", "seqs": 1, "rows": 8190, "kv_heads": 4, "head_dim": 256, "page": 32, "slot": 77},
        # Four conversations that have just begun, the smaller model's heads: latency.
        {"name": "attn_short", "kind": "attn", "seqs": 4, "shortest": 57, "longest": 700, "heads": 8, "kv_heads": 2, "head_dim": 256,
         "page": 16, "weights": False},
        # Sixteen conversations of unlike length whose caches are kept short by what is looked at.
        {"name": "attn_ragged", "kind": "attn", "seqs": 16, "shortest": 91, "longest": 16411, "heads": 24, "kv_heads": 4,
         "head_dim": 256, "page": 32, "weights": True},
        # Sixty-four of about the same length, head_dim 64.
        {"name": "attn_many", "kind": "attn", "seqs": 64, "shortest": 1800, "longest": 2300, "heads": 12, "kv_heads": 12,
         "head_dim": 64, "page": 64, "weights": False},
        # One long document at a length that no page divides, head_dim 128, its weights summed.
        {"name": "attn_32k", "kind": "attn", "seqs": 1, "shortest": 32771, "longest": 32771, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "page": 64, "weights": True},
        # The larger model's decode near the engine's longest context: the largest.
        {"name": "attn_262k", "kind": "attn", "seqs": 1, "shortest": 262000, "longest": 262000, "heads": 24, "kv_heads": 4,
         "head_dim": 256, "page": 64, "weights": False},
        # The steady state of a cache held at 2048 rows: each step one row more than that.
        {"name": "evict_step", "kind": "evict", "seqs": 16, "slots": 2049, "keep": 2048, "recent": 256, "kv_heads": 4,
         "head_dim": 256, "page": 16},
        # A long prompt brought down to an eighth.
        {"name": "evict_prompt", "kind": "evict", "seqs": 2, "slots": 32768, "keep": 4096, "recent": 512, "kv_heads": 4,
         "head_dim": 256, "page": 64},
        # The next token of one conversation, the usual settings.
        {"name": "sample_step", "kind": "sample", "rows": 1, "vocab": VOCAB, "temperature": 0.7, "top_k": 20, "top_p": 0.8,
         "min_p": 0.0, "coarse": False, "probs": False},
        # Sixteen conversations, each with its own settings, logits that were rounded to 16 bits (so many are alike).
        {"name": "sample_rows", "kind": "sample", "rows": 16, "vocab": VOCAB, "temperature": -1.0, "top_k": 0, "top_p": 1.0,
         "min_p": 0.0, "coarse": True, "probs": False},
        # Four guessed tokens' distributions for a check of them: no top-k, the probabilities written out.
        {"name": "sample_nucleus", "kind": "sample", "rows": 4, "vocab": VOCAB, "temperature": 1.0, "top_k": 0, "top_p": 0.95,
         "min_p": 0.001, "coarse": False, "probs": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(KINDS)
    if kind == "sample":
        c = {"kind": kind, "rows": _log(rng, 1, 16), "vocab": VOCAB if rng.random() < 0.5 else _log(rng, 500, VOCAB),
             "temperature": -1.0 if rng.random() < 0.3 else round(rng.uniform(0.3, 2.0), 3),
             "top_k": 0 if rng.random() < 0.4 else _log(rng, 1, 5000), "top_p": 1.0 if rng.random() < 0.3 else round(rng.uniform(0.3, 1.0), 4),
             "min_p": 0.0 if rng.random() < 0.5 else round(rng.uniform(0.0, 0.2), 4), "coarse": rng.random() < 0.4}
        c["probs"] = rng.random() < 0.5
        return c
    nh, nkv, hd = rng.choice(HEADS)
    page = rng.choice((16, 32, 64, 128, 256))
    if kind == "store":
        seqs = _log(rng, 1, 64)
        return {"kind": kind, "seqs": seqs, "rows": _log(rng, 1, max(1, 8192 // seqs)), "kv_heads": nkv, "head_dim": hd, "page": page,
                "slot": 0 if rng.random() < 0.25 else _log(rng, 1, 8192 // max(1, seqs // 8))}
    if kind == "attn":
        longest = _log(rng, 1, 262000)
        most = min(64, ELEMENTS // (longest * nkv * hd))
        return {"kind": kind, "seqs": _log(rng, 1, max(1, most)), "shortest": _log(rng, 1, longest), "longest": longest, "heads": nh,
                "kv_heads": nkv, "head_dim": hd, "page": page, "weights": rng.random() < 0.5}
    slots = _log(rng, 2, 65536)
    keep = max(1, slots - 1 if rng.random() < 0.3 else _log(rng, max(1, slots // 16), slots))
    most = min(16, ELEMENTS // 4 // (slots * nkv * hd))
    return {"kind": kind, "seqs": _log(rng, 1, max(1, most)), "slots": slots, "keep": keep, "recent": rng.randint(0, keep // 2),
            "kv_heads": nkv, "head_dim": hd, "page": page}


# ---------------------------------------------------------------- inputs

def _lens(case):
    """The sequences' lengths: evenly spread in their logarithm, mixed in order. Eviction: a few slots apart, the last one short."""
    n = case["seqs"]
    if case["kind"] == "evict":
        return [max(1, case["slots"] - 3 * i) if i < n - 1 or n < 3 else max(1, case["keep"] // 2) for i in range(n)]
    if case["kind"] == "store":
        return [max(0, case["slot"] - 37 * i) for i in range(n)]
    lo, hi = case["shortest"], case["longest"]
    out = [int(round(lo * (hi / lo) ** (i / max(1, n - 1)))) for i in range(n)] if n > 1 else [hi]
    return out[::2] + out[1::2][::-1]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(1000003 * (seed + 1) % (1 << 62))


def _normal(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def _width(case):
    """Pages of a table's row: room for the longest sequence and what comes."""
    most = max(_lens(case)) + (case["rows"] if case["kind"] == "store" else 0)
    return -(-most // case["page"]) + (1 if case["kind"] != "attn" else 0)


def _inputs(case, seed):
    g, k = _gen(seed), case["kind"]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    if k == "sample":
        r, v = case["rows"], case["vocab"]
        x = 3.0 * _normal(g, r, v)
        x.scatter_add_(1, torch.randint(0, v, (r, 12), generator=g, device="cuda"), 6.0 + 2.0 * _normal(g, r, 12))
        if case["coarse"]:
            x = x.bfloat16().float()
        z = np.random.default_rng(seed)
        s = np.zeros((r, 4), np.float32)
        top_k = np.full(r, case["top_k"], np.uint32)
        s[:, 0], s[:, 2], s[:, 3] = case["temperature"], case["top_p"], case["min_p"]
        if case["temperature"] < 0:             # each row its own
            s[:, 0] = z.choice([0.0, 0.3, 0.6, 0.7, 0.8, 1.0, 1.0, 1.2, 1.5], r)
            top_k[:] = z.choice([0, 0, 1, 5, 20, 40, 50, 64, 100, 1000], r)
            s[:, 2] = z.choice([1.0, 1.0, 0.5, 0.8, 0.9, 0.95, 0.99], r)
            s[:, 3] = z.choice([0.0, 0.0, 0.02, 0.05, 0.1], r)
        s[:, 1] = top_k.view(np.float32)
        return {"logits": x, "settings": torch.tensor(s.view(np.int32), device="cuda"),
                "u": torch.rand(r, generator=g, device="cuda")}
    n, nkv, hd, page, width = case["seqs"], case["kv_heads"], case["head_dim"], case["page"], _width(case)
    lens = _lens(case)
    pages = n * width + 3                       # no sequence shares one; three stay free
    t = {"table": torch.randperm(pages, generator=g, device="cuda")[:n * width].view(n, width).int()}
    t["kp"] = _normal(g, pages, page, nkv, hd, dtype=torch.float16) * torch.exp(0.5 * _normal(g, nkv, hd)).half()
    t["vp"] = _normal(g, pages, page, nkv, hd, dtype=torch.float16)
    if k == "store":
        t["rows"] = _normal(g, n, case["rows"], 2, nkv, hd)         # a projection's rows: keys, then values
        t["span"] = i32([[a, case["rows"] - (i % 3 if case["rows"] > 3 else 0), 5 * a // 4] for i, a in enumerate(lens)])
    else:
        t["lens"] = i32(lens)
    if k == "attn":
        t["q"] = _normal(g, n, case["heads"], hd)
    if k != "attn" or case["weights"]:
        w = torch.exp(2.0 * _normal(g, n, nkv, width * page))
        t["weight"] = torch.where(torch.rand(w.shape, generator=g, device="cuda") < 0.02, 0.0, w * 1e-3)
    if k != "attn":
        gaps = torch.randint(1, 3, (n, nkv, width * page), generator=g, device="cuda", dtype=torch.int32)
        t["pos"] = gaps.cumsum(dim=2).int()     # rows were evicted before, so positions have gaps
    return t


# ---------------------------------------------------------------- what a program holds

class _Dev:
    """A tensor's memory, from element `off` on, as a buffer handle."""

    def __init__(self, gpu, t, off=0):
        import surge_amd as S
        self.t, self.free = t, S.lib().sg_gpu_buf_free
        self.handle = C.c_void_p()
        S.check(S.lib().sg_gpu_wrap_device(gpu.handle, t.data_ptr() + off * t.element_size(),
                                           (t.numel() - off) * t.element_size(), C.byref(self.handle)))

    def __del__(self):
        if self.handle:
            self.free(self.handle)


_one_gpu = None


def _gpu():
    global _one_gpu
    if _one_gpu is None:
        import surge_amd as S
        _one_gpu = S.Gpu()
    return _one_gpu


def prepare(case, seed):
    t, k = _inputs(case, seed), case["kind"]
    if k == "sample":
        t["token"] = torch.zeros(case["rows"], device="cuda", dtype=torch.int32)
        if case["probs"]:
            t["probs"] = torch.empty_like(t["logits"])
    elif k == "attn":
        t["out"] = torch.empty_like(t["q"])
        if case["weights"]:
            t["weight_out"] = t["weight"].clone()
    elif k == "evict":
        t["weight_out"], t["pos_out"] = t["weight"].clone(), t["pos"].clone()
    state = {"case": case, "t": t}
    if own:
        import surge_amd as S
        gpu = _gpu()
        b = {n: _Dev(gpu, x) for n, x in t.items()}
        state["gpu"], state["b"] = gpu, b
        if k == "sample":
            state["p"] = [case["vocab"], case["rows"]]
        else:
            nkv, hd, page, n, width = case["kv_heads"], case["head_dim"], case["page"], case["seqs"], _width(case)
            if k == "store":
                b["vrows"] = _Dev(gpu, t["rows"], nkv * hd)
                state["p"] = [nkv, hd, page, n, width, case["rows"], 2 * nkv * hd]
            elif k == "attn":
                state["p"] = [case["heads"], nkv, hd, page, n, width, hd, S.fbits(1 / math.sqrt(hd))]
            else:
                state["p"] = [nkv, hd, page, n, width, case["keep"], case["recent"]]
    return state


# ---------------------------------------------------------------- one pass

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    k, g, t, b, p = state["case"]["kind"], state["gpu"], state["t"], state["b"], state["p"]
    if k == "store":
        g.page_store(b["rows"], b["vrows"], b["kp"], b["vp"], b["table"], b["span"], b["weight"], b["pos"], p)
    elif k == "attn":
        g.attn_paged(b["q"], b["kp"], b["vp"], b["table"], b["lens"], b.get("weight"), b.get("weight_out"), b["out"], p)
    elif k == "evict":
        g.page_evict(b["kp"], b["vp"], b["table"], b["lens"], b["weight"], b["pos"], b["weight_out"], b["pos_out"], p)
    else:
        g.sample(b["logits"], b["settings"], b["u"], b["token"], b.get("probs"), p)
    return _outputs(k, t)


def _outputs(k, t):
    names = {"store": ("kp", "vp", "weight", "pos"), "attn": ("out", "weight_out"), "evict": ("kp", "vp", "weight_out", "pos_out"),
             "sample": ("token", "probs")}[k]
    return {n: t[n] for n in names if n in t}


def _run_plain(state):
    c, t = state["case"], state["t"]
    {"store": _store_plain, "attn": _attn_plain, "evict": _evict_plain, "sample": _sample_plain}[c["kind"]](c, t)
    return _outputs(c["kind"], t)


def _store_plain(c, t):
    n, nkv, hd, page, rows = c["seqs"], c["kv_heads"], c["head_dim"], c["page"], c["rows"]
    i = torch.arange(rows, device="cuda")
    slot = t["span"][:, :1].long() + i
    s, i = (i < t["span"][:, 1:2]).nonzero(as_tuple=True)
    slot = slot[s, i]
    at = t["table"][s, slot // page].long() * page + slot % page
    for half, pool in enumerate((t["kp"], t["vp"])):
        pool.view(-1, nkv, hd)[at] = t["rows"][s, i, half].half()
    t["weight"][s, :, slot] = 0.0
    t["pos"][s, :, slot] = (t["span"][s, 2] + i).int()[:, None]


def _attn_plain(c, t):
    n, nh, nkv, hd = c["seqs"], c["heads"], c["kv_heads"], c["head_dim"]
    page, group = c["page"], nh // nkv
    tab = t["table"].long()
    seq = tab.shape[1] * page
    kf = t["kp"][tab].view(n, seq, nkv, hd).permute(0, 2, 3, 1).float().contiguous()
    s = torch.matmul(t["q"].view(n, nkv, group, hd), kf) * (1 / math.sqrt(hd))
    del kf
    s.masked_fill_(torch.arange(seq, device="cuda") >= t["lens"].long()[:, None, None, None], -math.inf)
    p = torch.exp(s - s.amax(dim=3, keepdim=True))
    p /= p.sum(dim=3, keepdim=True)
    vf = t["vp"][tab].view(n, seq, nkv, hd).permute(0, 2, 1, 3).float().contiguous()
    t["out"].view(n, nkv, group, hd)[...] = torch.matmul(p, vf)
    if c["weights"]:
        t["weight_out"][...] = t["weight"] + p.sum(dim=2)


def _evict_plain(c, t):
    nkv, hd, page, keep = c["kv_heads"], c["head_dim"], c["page"], c["keep"]
    w, pos, ln = t["weight"], t["pos"], t["lens"].long()[:, None, None]
    cap = w.shape[2]
    slot = torch.arange(cap, device="cuda")
    held = slot < ln
    last = torch.where(held, pos, -2 ** 31).amax(dim=2, keepdim=True).long()
    rank_by = torch.where(pos > last - c["recent"], math.inf, w).masked_fill_(~held, -math.inf)
    order = torch.argsort(rank_by, dim=2, descending=True, stable=True)     # alike: the lower slot first
    kept = torch.zeros_like(held.expand_as(w)).scatter_(2, order[:, :, :keep], True) & held
    hole = ~kept[:, :, :keep] & held[:, :, :keep]
    mover = kept.clone()
    mover[:, :, :keep] = False
    movers = torch.argsort((~mover).int(), dim=2, stable=True)              # the moved rows' slots, in order
    nth = hole.cumsum(dim=2) - 1
    src = torch.where(hole, movers.gather(2, nth.clamp_min(0)), slot[:keep])
    within = (slot[:keep] < ln).expand_as(src)
    for old, new in ((w, t["weight_out"]), (pos, t["pos_out"])):
        new[:, :, :keep] = torch.where(within, old.gather(2, src), new[:, :, :keep])
    s, h, d = hole.nonzero(as_tuple=True)
    f = src[s, h, d]
    row = lambda x: t["table"][s, x // page].long() * page + x % page
    to, of = row(d), row(f)
    for pool in (t["kp"], t["vp"]):
        flat = pool.view(-1, nkv, hd)
        flat[to, h] = flat[of, h]


def _sample_plain(c, t):
    x, s = t["logits"], t["settings"]
    v = x.shape[1]
    temp, top_p, min_p = (s[:, i:i + 1].contiguous().view(torch.float32).double() for i in (0, 2, 3))
    top_k = s[:, 1:2].long()
    greedy = ~(temp > 0)
    top_k = torch.where(greedy, 1, torch.where(top_k > 0, top_k, v))
    ok = x > -math.inf
    x = torch.where(ok, x, -math.inf)
    z = (x.double() - x.amax(dim=1, keepdim=True).double()) / torch.where(greedy, 1.0, temp)
    w = torch.exp(z) * ok
    order = torch.argsort(x, dim=1, descending=True, stable=True)           # alike: the lower id first
    first = torch.arange(v, device="cuda") < top_k
    ws = w.gather(1, order) * first
    cum = ws.cumsum(dim=1)
    before = torch.nn.functional.pad(cum[:, :-1], (1, 0))
    first &= (before < top_p * cum[:, -1:]) | (top_p >= 1) | (torch.arange(v, device="cuda") == 0)
    first &= ws >= min_p
    kept = torch.zeros_like(ok).scatter_(1, order, first) & ok
    w = w * kept
    cum = w.cumsum(dim=1)
    total = cum[:, -1:]
    i = torch.arange(v, device="cuda")
    t["token"][...] = torch.where(kept & (cum > t["u"].double()[:, None] * total), i, v).amin(dim=1).int()
    if "probs" in t:
        t["probs"][...] = w / total


# ---------------------------------------------------------------- the work of one pass

def work(case):
    k = case["kind"]
    if k == "sample":
        e = case["rows"] * case["vocab"]
        return {"bytes": 4 * e * (2 if case["probs"] else 1) + 24 * case["rows"], "flops": 6 * e}
    nkv, hd = case["kv_heads"], case["head_dim"]
    if k == "store":
        n = case["rows"] * case["seqs"]
        return {"bytes": n * nkv * (2 * hd * 6 + 8), "flops": 2 * n * nkv * hd}
    lens = _lens(case)
    if k == "attn":
        nh, total = case["heads"], sum(lens)
        return {"bytes": 4 * total * nkv * hd + 8 * case["seqs"] * nh * hd + (8 * total * nkv if case["weights"] else 0),
                "flops": 4 * total * nh * hd}
    keep = case["keep"]
    moved = sum((n - keep) * (case["recent"] / n + (1 - case["recent"] / n) * keep / n) for n in lens if n > keep)
    return {"bytes": int(nkv * (8 * moved * hd + 8 * sum(lens) + 8 * sum(min(n, keep) for n in lens))), "flops": 2 * nkv * sum(lens)}


# ---------------------------------------------------------------- the same in 64 bits, from the definitions

def exact(case, seed):
    t, k = _inputs(case, seed), case["kind"]
    f8 = np.float64
    if k == "sample":
        return _sample_exact(case, t)
    n, nkv, hd, page = case["seqs"], case["kv_heads"], case["head_dim"], case["page"]
    lens = _lens(case)
    if k == "attn":
        return _attn_exact(case, t, lens)
    table, kp, vp = (t[x].cpu().numpy() for x in ("table", "kp", "vp"))
    weight, pos = t["weight"].cpu().numpy(), t["pos"].cpu().numpy()
    cell = lambda s, j: (table[s, j // page], j % page)
    if k == "store":
        rows, span = t["rows"].cpu().numpy(), t["span"].cpu().numpy()
        for s in range(n):
            a, m, p = (int(x) for x in span[s])
            j = np.arange(a, a + m)
            kp[cell(s, j)], vp[cell(s, j)] = rows[s, :m, 0].astype(np.float16), rows[s, :m, 1].astype(np.float16)
            weight[s, :, j], pos[s, :, j] = 0.0, np.arange(p, p + m)[:, None]
        return {"kp": kp, "vp": vp, "weight": weight.astype(f8), "pos": pos}
    keep = case["keep"]
    wo, po = weight.copy(), pos.copy()
    for s in range(n):
        m = lens[s]
        if m <= keep:
            continue
        for h in range(nkv):
            w, p = weight[s, h, :m], pos[s, h, :m].astype(np.int64)
            old = p <= p.max() - case["recent"]
            best = np.lexsort((np.arange(m), -w.astype(f8), old))[:keep]
            holes = np.setdiff1d(np.arange(keep), best)
            movers = np.sort(best[best >= keep])
            wo[s, h, holes], po[s, h, holes] = w[movers], p[movers]
            (a, b), (x, y) = cell(s, holes), cell(s, movers)
            kp[a, b, h], vp[a, b, h] = kp[x, y, h], vp[x, y, h]
    return {"kp": kp, "vp": vp, "weight_out": wo.astype(f8), "pos_out": po}


def _attn_exact(case, t, lens):
    n, nh, nkv, hd, page = (case[x] for x in ("seqs", "heads", "kv_heads", "head_dim", "page"))
    group = nh // nkv
    q = t["q"].double().view(n, nkv, group, hd)
    out = torch.zeros(n, nkv, group, hd, dtype=torch.float64, device="cuda")
    wo = t["weight"].double() if case["weights"] else None
    for s in range(n):
        own_pages = t["table"][s, :-(-lens[s] // page)].long()
        for h in range(nkv):
            kd = t["kp"][own_pages, :, h].reshape(-1, hd)[:lens[s]].double()
            vd = t["vp"][own_pages, :, h].reshape(-1, hd)[:lens[s]].double()
            p = torch.softmax(torch.mm(q[s, h], kd.t().contiguous()) / math.sqrt(hd), dim=1)
            out[s, h] = torch.mm(p, vd)
            if wo is not None:
                wo[s, h, :lens[s]] += p.sum(dim=0)
    r = {"out": out.view(n, nh, hd).cpu().numpy()}
    if wo is not None:
        r["weight_out"] = wo.cpu().numpy()
    return r


def _sample_exact(case, t):
    logits, u = t["logits"].cpu().numpy(), t["u"].cpu().numpy()
    s = t["settings"].cpu().numpy()
    f = np.ascontiguousarray(s).view(np.float32)
    token, probs = np.zeros(len(logits), np.int32), np.zeros(logits.shape)
    for r, x in enumerate(logits.astype(np.float64)):
        temp, k, p, low = float(f[r, 0]), int(s[r, 1]), float(f[r, 2]), float(f[r, 3])
        if not temp > 0:
            temp, k = 1.0, 1
        ids = np.argsort(-x, kind="stable")[:k or len(x)]
        w = np.exp((x[ids] - x[ids[0]]) / temp)
        cum = np.cumsum(w.astype(np.longdouble))
        m = len(ids) if p >= 1 else max(1, int(np.searchsorted(cum, p * cum[-1], side="left")) + 1)
        ids, w = ids[:m], w[:m]
        ids = np.sort(ids[w >= low])
        w = np.exp((x[ids] - x.max()) / temp)
        cum = np.cumsum(w.astype(np.longdouble))
        token[r] = ids[min(int(np.searchsorted(cum, float(u[r]) * cum[-1], side="right")), len(ids) - 1)]
        probs[r, ids] = w / float(cum[-1])
    return {"token": token, "probs": probs} if case["probs"] else {"token": token}
