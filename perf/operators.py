"""Timed cases of the dense serving operators: attention over whole prompts (causal, grouped
heads, packed sequences), attention of one new token over a paged K / V cache, writing new
K / V rows into the cache's pages, and forking / compacting those pages.

``run`` computes a case in elementary torch operations (32-bit arithmetic, one rounding at
the end), or, where ``own`` is set, through ``mzoo_b200.gqa_attn`` and ``mzoo_b200.kv_pages``.
``exact`` states the same results in 64 bits.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
GOLDEN = 0.6180339887498949


def listed():
    return [
        # one short chat turn, the 16 heads on 1 KV head of the window configuration: latency
        dict(name="prefill short", op="prefill", dtype="bf16", hq=16, hkv=1, d=128, seqs=1, lo=33, hi=33, past_lo=0,
             past_hi=0, fused=True),
        # a scheduler's packed batch of unequal prompts, q / k / v as slices of one projection
        dict(name="prefill packed", op="prefill", dtype="bf16", hq=32, hkv=8, d=128, seqs=9, lo=1, hi=2047, past_lo=0,
             past_hi=0, fused=True),
        # the next chunk of long prompts: 6 query heads to a KV head, earlier keys in front
        dict(name="prefill chunk", op="prefill", dtype="fp16", hq=24, hkv=4, d=64, seqs=2, lo=777, hi=1100,
             past_lo=3001, past_hi=5000, fused=False),
        # one long document
        dict(name="prefill long", op="prefill", dtype="bf16", hq=16, hkv=2, d=128, seqs=1, lo=16384, hi=16384,
             past_lo=0, past_hi=0, fused=False),
        # the first tokens of one conversation: latency
        dict(name="decode short", op="decode", dtype="bf16", hq=32, hkv=8, d=128, page=16, seqs=1, lo=77, hi=77),
        # a full serving batch of unequal contexts
        dict(name="decode batch", op="decode", dtype="bf16", hq=32, hkv=8, d=128, page=64, seqs=64, lo=512, hi=16384),
        # one long context alone on the GPU
        dict(name="decode long", op="decode", dtype="bf16", hq=32, hkv=8, d=128, page=64, seqs=1, lo=131001, hi=131001),
        # one KV head, empty slots among the sequences
        dict(name="decode one kv head", op="decode", dtype="fp16", hq=16, hkv=1, d=64, page=32, seqs=37, lo=0, hi=4096),
        # the cache write of one decode step
        dict(name="append step", op="append", dtype="bf16", hkv=8, d=128, page=64, seqs=128, lo=1, hi=1, past_lo=100,
             past_hi=3000),
        # the cache write of a packed batch of prompts
        dict(name="append prompts", op="append", dtype="bf16", hkv=8, d=128, page=64, seqs=9, lo=40, hi=4095,
             past_lo=0, past_hi=200),
        # parallel sampling: eight answers to each of eight prompts, K and V of four layers
        dict(name="fork samples", op="fork", dtype="bf16", hkv=8, d=128, page=32, pools=8, seqs=8, copies=8, lo=700,
             hi=4100, spare=600),
        # half of the pages are left after requests finished: the live ones move to the front
        dict(name="compact half", op="compact", dtype="bf16", hkv=8, d=128, page=32, pools=2, pages=8192, live=0.5,
             width=256),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["prefill", "prefill", "decode", "decode", "append", "fork", "compact"])
    c = dict(op=op, dtype=rng.choice(["bf16", "fp16"]), hkv=rng.choice([1, 2, 4, 8]), d=rng.choice([64, 96, 128]))
    if op == "prefill":
        while True:
            c.update(hq=c["hkv"] * rng.choice([1, 2, 3, 4, 6, 8, 16]), seqs=_log(rng, 1, 16), hi=_log(rng, 1, 12000))
            c.update(lo=rng.randint(1, c["hi"]), past_hi=rng.choice([0, _log(rng, 1, 6000)]))
            c.update(past_lo=rng.randint(0, c["past_hi"]), fused=c["past_hi"] == 0 and rng.random() < 0.5)
            if c["seqs"] * c["hq"] * c["hi"] * (c["hi"] + c["past_hi"]) <= 16 * 16384 ** 2 // 2 and c["hq"] <= 64:
                return c
    if op == "decode":
        while True:
            c.update(hq=c["hkv"] * rng.choice([1, 2, 3, 4, 6, 8, 16]), page=rng.choice([16, 32, 64, 128]),
                     seqs=_log(rng, 1, 256), hi=_log(rng, 1, 131072))
            c.update(lo=rng.randint(0, c["hi"]))
            if c["seqs"] * c["hi"] * c["hkv"] * c["d"] <= 64 * 8192 * 8 * 128 and c["hq"] <= 64:
                return c
    if op == "append":
        c.update(page=rng.choice([16, 32, 64, 128]), seqs=_log(rng, 1, 128), hi=_log(rng, 1, 256))
        c.update(lo=rng.randint(0, c["hi"]), past_hi=_log(rng, 1, 2000))
        c.update(past_lo=rng.randint(0, c["past_hi"]))
        return c
    if op == "fork":
        c.update(page=rng.choice([16, 32, 64]), pools=rng.choice([2, 4, 8]), seqs=_log(rng, 1, 8), copies=_log(rng, 1, 8),
                 hi=_log(rng, 1, 4000), spare=rng.randint(100, 700))
        c.update(lo=rng.randint(0, c["hi"]))
        return c
    c.update(page=rng.choice([16, 32]), pools=2, pages=_log(rng, 17, 8000), live=round(rng.uniform(0.05, 0.95), 3),
             width=rng.randint(1, 200))
    return c


# ------------------------------------------------------------------ sizes of a case

def _spread(n, lo, hi):
    """n whole numbers from lo to hi, evenly spread and in no order (hi alone for one)."""
    if n == 1:
        return [hi]
    got = [int(round(lo + ((i * GOLDEN) % 1.0) * (hi - lo))) for i in range(n)]
    got[n // 2] = hi
    return got


def _lens(c):
    """(new tokens, tokens before them) of each sequence."""
    new = _spread(c["seqs"], c["lo"], c["hi"])
    return new, _spread(c["seqs"], c.get("past_lo", 0), c.get("past_hi", 0))


def _starts(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return at


def work(c):
    new, past = _lens(c) if "seqs" in c else ([], [])
    if c["op"] == "prefill":
        tq, tk = sum(new), sum(new) + sum(past)
        pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(new, past))
        return {"bytes": 2 * c["d"] * (2 * tq * c["hq"] + 2 * tk * c["hkv"]) + 4 * tq * c["hq"],
                "flops": 4 * c["d"] * c["hq"] * pairs}
    if c["op"] == "decode":
        t = sum(new)
        return {"bytes": 4 * t * c["hkv"] * c["d"] + 4 * c["seqs"] * c["hq"] * (c["d"] + 1) + 4 * -(-t // c["page"]),
                "flops": 4 * c["d"] * c["hq"] * t}
    row = 2 * c["hkv"] * c["d"]
    if c["op"] == "append":
        return {"bytes": 4 * row * sum(new) + 12 * c["seqs"], "flops": 0}
    if c["op"] == "fork":
        tails = c["copies"] * sum(n % c["page"] > 0 for n in new)
        return {"bytes": 2 * tails * c["pools"] * c["page"] * row + 16 * c["copies"] * sum(-(-n // c["page"]) for n in new),
                "flops": 0}
    live = _live(c)
    return {"bytes": 2 * live * (c["pages"] - live) // c["pages"] * c["pools"] * c["page"] * row + 16 * c["pages"], "flops": 0}


def _live(c):
    return max(1, min(c["pages"] - 1, int(c["live"] * c["pages"])))


# ------------------------------------------------------------------ inputs

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, dtype, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _pool(g, dtype, *shape):
    """Pages' contents; filled a part at a time, since the 32-bit draw is twice as large."""
    out = torch.empty(*shape, device="cuda", dtype=dtype)
    for part in out.split(max(1, (1 << 27) // out[0].numel())):
        part.copy_(torch.randn(part.shape, generator=g, device="cuda", dtype=torch.float32))
    return out


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _table(g, lens, page, pages, width):
    """Page tables over a random order of the pages, -1 behind each sequence's last page."""
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    need = torch.tensor([-(-n // page) for n in lens], device="cuda")
    first = torch.cumsum(need, 0) - need
    cols = torch.arange(width, device="cuda")
    used = cols[None, :] < need[:, None]
    at = (first[:, None] + cols[None, :]).clamp(max=pages - 1)
    return torch.where(used, order[at], torch.full_like(order[at], -1)), used, order


def prepare(c, seed):
    g, dt = _generator(seed), DTYPES[c["dtype"]]
    s = {"case": c, "op": c["op"]}
    if c["op"] == "prefill":
        new, past = _lens(c)
        keys = [n + p for n, p in zip(new, past)]
        tq, tk = sum(new), sum(keys)
        if c["fused"]:  # one projection's output [tokens, (hq + 2 hkv) d]: q, k and v are views of it
            qkv = _normal(g, dt, tq, c["hq"] + 2 * c["hkv"], c["d"])
            q, k, v = qkv.split([c["hq"], c["hkv"], c["hkv"]], dim=1)
        else:
            q, k, v = (_normal(g, dt, t, h, c["d"]) for t, h in ((tq, c["hq"]), (tk, c["hkv"]), (tk, c["hkv"])))
        return s | {"q": q, "k": k, "v": v, "cu_q": _int(_starts(new)), "cu_k": _int(_starts(keys)), "max_q": max(new),
                    "max_k": max(keys)}
    if c["op"] == "decode":
        lens, page = _lens(c)[0], c["page"]
        need = sum(-(-n // page) for n in lens)
        pages, width = need + need // 16 + 2, max(1, -(-max(lens) // page))
        shape = (pages, c["hkv"], page, c["d"])
        return s | {"q": _normal(g, dt, c["seqs"], c["hq"], c["d"]), "k_pages": _pool(g, dt, *shape),
                    "v_pages": _pool(g, dt, *shape), "table": _table(g, lens, page, pages, width)[0], "lens": _int(lens)}
    if c["op"] == "append":
        new, past = _lens(c)
        page, total = c["page"], [n + p for n, p in zip(new, past)]
        need = sum(-(-n // page) for n in total)
        pages, shape = need + 8, (need + 8, c["hkv"], page, c["d"])
        return s | {"k": _normal(g, dt, sum(new), c["hkv"], c["d"]), "v": _normal(g, dt, sum(new), c["hkv"], c["d"]),
                    "k_pages": _pool(g, dt, *shape), "v_pages": _pool(g, dt, *shape), "starts": _int(past),
                    "table": _table(g, total, page, pages, max(1, -(-max(total) // page)))[0], "cu": _int(_starts(new))}
    if c["op"] == "fork":
        lens, page, n = _lens(c)[0], c["page"], c["seqs"]
        need = sum(-(-x // page) for x in lens)
        pages = need + c["spare"]
        table, used, order = _table(g, lens, page, pages, max(1, -(-max(lens) // page)))
        slots = n * (1 + c["copies"])
        full = torch.full((slots, table.shape[1]), -1, dtype=torch.int32, device="cuda")
        full[:n] = table
        refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
        refs[order[:need].long()] = 1
        parents = [i for i in range(n) for _ in range(c["copies"])]
        return s | {"pools": [_pool(g, dt, pages, c["hkv"], page, c["d"]) for _ in range(c["pools"])], "table": full,
                    "lens": _int(lens + [0] * (slots - n)), "refs": refs, "src": _int(parents),
                    "dst": _int(list(range(n, slots)))}
    pages, live, width = c["pages"], _live(c), c["width"]
    order = torch.randperm(pages, generator=g, device="cuda")[:live].to(torch.int32)
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[order.long()] = torch.randint(1, 4, (live,), generator=g, device="cuda", dtype=torch.int32)
    rows = -(-live // width)
    table = torch.full((rows * width,), -1, dtype=torch.int32, device="cuda")
    table[:live] = order
    return s | {"pools": [_pool(g, dt, pages, c["hkv"], c["page"], c["d"]) for _ in range(c["pools"])],
                "table": table.view(rows, width), "refs": refs}


# ------------------------------------------------------------------ one pass

def run(s):
    return (_own if own else _plain)[s["op"]](s)


def _softmax_rows(scores, seen):
    """exp(scores - row maximum) with nothing where `seen` is false, the row sums and the
    logarithm of the summed exponentials; a row that sees nothing has sum 0 and lse -inf."""
    scores.masked_fill_(~seen, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    return p, total, (top + total.log()).squeeze(-1)


def _plain_prefill(s):
    c, cu_q, cu_k = s["case"], s["cu_q"].long(), s["cu_k"].long()
    n, hkv, grp, d = c["seqs"], c["hkv"], c["hq"] // c["hkv"], c["d"]
    iq, ik = torch.arange(s["max_q"], device="cuda"), torch.arange(s["max_k"], device="cuda")
    len_q, len_k = cu_q[1:] - cu_q[:-1], cu_k[1:] - cu_k[:-1]
    at_q = (cu_q[:-1, None] + iq).clamp(max=s["q"].shape[0] - 1)
    at_k = (cu_k[:-1, None] + ik).clamp(max=s["k"].shape[0] - 1)
    q = s["q"][at_q].float().view(n, -1, hkv, grp, d)
    k, v = s["k"][at_k].float(), s["v"][at_k].float()
    scores = torch.einsum("bqhgd,bkhd->bhgqk", q, k).mul_(d ** -0.5)
    last = iq[None, :] + (len_k - len_q)[:, None]  # the last key that each token sees
    seen = (ik <= last[:, :, None]) & (ik < len_k[:, None, None])
    p, total, lse = _softmax_rows(scores, seen[:, None, None])
    o = torch.einsum("bhgqk,bkhd->bhgqd", p, v) / torch.where(total > 0, total, torch.ones_like(total))
    seq = torch.searchsorted(cu_q, torch.arange(s["q"].shape[0], device="cuda"), right=True) - 1
    at = torch.arange(s["q"].shape[0], device="cuda") - cu_q[seq]
    return {"o": o.permute(0, 3, 1, 2, 4)[seq, at].reshape(-1, c["hq"], d).to(s["q"].dtype),
            "lse": lse.permute(0, 3, 1, 2)[seq, at].reshape(-1, c["hq"])}


def _plain_decode(s):
    c, lens = s["case"], s["lens"].long()
    n, hkv, grp, d = c["seqs"], c["hkv"], c["hq"] // c["hkv"], c["d"]
    table = s["table"].long().clamp(min=0)
    q = s["q"].float().view(n, hkv, grp, d)
    k = s["k_pages"][table].float().permute(0, 2, 1, 3, 4).reshape(n, hkv, -1, d)
    scores = torch.matmul(q, k.transpose(-1, -2)).mul_(d ** -0.5)
    del k
    seen = torch.arange(scores.shape[-1], device="cuda") < lens[:, None]
    p, total, lse = _softmax_rows(scores, seen[:, None, None])
    v = s["v_pages"][table].float().permute(0, 2, 1, 3, 4).reshape(n, hkv, -1, d)
    o = torch.matmul(p, v) / torch.where(total > 0, total, torch.ones_like(total))
    return {"o": o.reshape(n, -1, d).to(s["q"].dtype), "lse": lse.reshape(n, -1)}


def _plain_append(s):
    cu, page = s["cu"].long(), s["case"]["page"]
    i = torch.arange(s["k"].shape[0], device="cuda")
    seq = torch.searchsorted(cu, i, right=True) - 1
    pos = s["starts"].long()[seq] + i - cu[seq]
    at, slot = s["table"].long()[seq, pos // page], pos % page
    s["k_pages"][at, :, slot] = s["k"]
    s["v_pages"][at, :, slot] = s["v"]
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _plain_fork(s):
    table, lens, refs, page = s["table"], s["lens"], s["refs"], s["case"]["page"]
    src, dst = s["src"].long(), s["dst"].long()
    old = table[dst]
    refs.scatter_add_(0, old.clamp(min=0).long().flatten(), -(old >= 0).to(refs.dtype).flatten())
    n = lens[src]
    row, full = table[src], (n // page).long()
    shared = torch.arange(table.shape[1], device="cuda") < full[:, None]
    refs.scatter_add_(0, row.clamp(min=0).long().flatten(), shared.to(refs.dtype).flatten())
    tail = torch.nonzero(n % page)[:, 0]  # the copies whose last page is not full
    new = torch.nonzero(refs == 0)[:tail.numel(), 0]
    refs[new] = 1
    row_new = torch.where(shared, row, torch.full_like(row, -1))
    row_new[tail, full[tail]] = new.to(torch.int32)
    table[dst], lens[dst] = row_new, n
    of = row[tail, full[tail]].long()
    for pool in s["pools"]:
        pool[new] = pool[of]
    return {"table": table, "lens": lens, "refs": refs, "pools": s["pools"]}


def _plain_compact(s):
    refs, table = s["refs"], s["table"]
    live = refs > 0
    n = live.sum()
    at = torch.arange(refs.numel(), device="cuda")
    moved, hole = torch.nonzero(live & (at >= n))[:, 0], torch.nonzero(~live & (at < n))[:, 0]
    to = at.clone()
    to[moved] = hole
    for pool in s["pools"]:
        pool[hole] = pool[moved]
    new_refs = torch.where(at < n, refs, torch.zeros_like(refs))
    new_refs[hole] = refs[moved]
    new_table = torch.where(table >= 0, to[table.clamp(min=0).long()].to(torch.int32), table)
    return {"table": new_table, "refs": new_refs, "pools": s["pools"]}


def _own_prefill(s):
    from mzoo_b200 import gqa_attn
    o, lse = gqa_attn.prefill(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"])
    return {"o": o, "lse": lse}


def _own_decode(s):
    from mzoo_b200 import gqa_attn
    o, lse = gqa_attn.decode(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"])
    return {"o": o, "lse": lse}


def _own_append(s):
    from mzoo_b200 import kv_pages
    kv_pages.append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["starts"], s["cu"])
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _own_fork(s):
    from mzoo_b200 import kv_pages
    kv_pages.fork(s["pools"], s["table"], s["lens"], s["refs"], s["src"], s["dst"], page_size=s["case"]["page"])
    return {"table": s["table"], "lens": s["lens"], "refs": s["refs"], "pools": s["pools"]}


def _own_compact(s):
    from mzoo_b200 import kv_pages
    table, refs = kv_pages.compact(s["pools"], s["table"], s["refs"])
    return {"table": table, "refs": refs, "pools": s["pools"]}


_plain = {"prefill": _plain_prefill, "decode": _plain_decode, "append": _plain_append, "fork": _plain_fork,
          "compact": _plain_compact}
_own = {"prefill": _own_prefill, "decode": _own_decode, "append": _own_append, "fork": _own_fork,
        "compact": _own_compact}


# ------------------------------------------------------------------ the definition in 64 bits

def _attend64(q, k, v, seen):
    """softmax(q k^T / sqrt(d)) v over the keys `seen`, and the log-sum-exp, one head in doubles."""
    x = (q @ k.T / math.sqrt(q.shape[-1])).masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(x, -1)
    p = torch.exp(x - torch.where(torch.isinf(lse), torch.zeros_like(lse), lse)[:, None])
    return p @ v, lse


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "prefill":
        q, k, v = (s[x].double() for x in "qkv")
        o, lse = torch.zeros_like(q), torch.zeros(q.shape[:2], device="cuda", dtype=torch.float64)
        new, past = _lens(c)
        a = b = 0
        for n, p in zip(new, past):
            i, j = torch.arange(n, device="cuda")[:, None], torch.arange(n + p, device="cuda")[None, :]
            for h in range(c["hq"]):
                kh = h // (c["hq"] // c["hkv"])
                o[a:a + n, h], lse[a:a + n, h] = _attend64(q[a:a + n, h], k[b:b + n + p, kh], v[b:b + n + p, kh], j <= i + p)
            a, b = a + n, b + n + p
        return {"o": o, "lse": lse}
    if c["op"] == "decode":
        q, grp = s["q"].double(), c["hq"] // c["hkv"]
        o, lse = torch.zeros_like(q), torch.full(q.shape[:2], -math.inf, device="cuda", dtype=torch.float64)
        for b, n in enumerate(_lens(c)[0]):
            if n:
                ids = s["table"][b, :-(-n // c["page"])].long()
                k, v = (s[x][ids].transpose(0, 1).flatten(1, 2)[:, :n].double() for x in ("k_pages", "v_pages"))
                x = torch.einsum("hgd,hkd->hgk", q[b].view(-1, grp, c["d"]), k) / math.sqrt(c["d"])
                lse[b] = torch.logsumexp(x, -1).flatten()
                o[b] = torch.einsum("hgk,hkd->hgd", torch.softmax(x, -1), v).flatten(0, 1)
        return {"o": o, "lse": lse}
    if c["op"] == "append":
        k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
        table, (new, past), at = s["table"].tolist(), _lens(c), 0
        for b, (n, p) in enumerate(zip(new, past)):
            done = 0
            while done < n:  # a page's share at a time
                page, slot = divmod(p + done, c["page"])
                m = min(n - done, c["page"] - slot)
                for pool, x in ((k_pages, s["k"]), (v_pages, s["v"])):
                    pool[table[b][page], :, slot:slot + m] = x[at + done:at + done + m].transpose(0, 1).double()
                done += m
            at += n
        return {"k_pages": k_pages, "v_pages": v_pages}
    table, refs = s["table"].tolist(), s["refs"].tolist()
    if c["op"] == "fork":
        lens, copied = s["lens"].tolist(), []
        pairs = list(zip(s["src"].tolist(), s["dst"].tolist()))
        for a, b in pairs:
            table[b], lens[b] = [p if i < lens[a] // c["page"] else -1 for i, p in enumerate(table[a])], lens[a]
            for p in table[b]:
                if p >= 0:
                    refs[p] += 1
        free = (p for p, r in enumerate(list(refs)) if r == 0)
        for a, b in pairs:
            if lens[a] % c["page"]:
                p, i = next(free), lens[a] // c["page"]
                table[b][i], refs[p] = p, 1
                copied.append((table[a][i], p))
        out = {"table": _int(table), "lens": _int(lens), "refs": _int(refs)}
    else:
        n, copied = sum(r > 0 for r in refs), []
        holes, to = [p for p in range(n) if refs[p] == 0], {}
        for p in range(n, len(refs)):
            if refs[p] > 0:
                to[p] = holes[len(copied)]
                copied.append((p, to[p]))
                refs[to[p]], refs[p] = refs[p], 0
        out = {"table": _int([[to.get(p, p) for p in row] for row in table]), "refs": _int(refs)}
    pools = [pool.double() for pool in s["pools"]]
    if copied:
        a, b = (torch.tensor(x, device="cuda") for x in zip(*copied))
        for pool in pools:
            pool[b] = pool[a]
    return out | {"pools": pools}
