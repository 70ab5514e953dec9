"""The attention and key-value cache operators: cases, plain forms and exact values.

Four operators that a program serving a transformer block needs around the
block's contractions: attention over a packed prompt, attention of one new
token over a paged key-value cache, writing new keys and values into the
cache's pages, and the management of those pages (fork, compact). `run` makes
one pass: in the plain form (elementary torch operations in 32 bits) or, with
`own`, through tosa_b200.attention.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # the next turn of a chat: a short question whose earlier turns are already keys; latency counts
        dict(name="prompt turn", op="prompt", dtype="f16", seqs=1, shortest=61, longest=61, prefix=129, mix=1,
             q_heads=8, kv_heads=2, head_dim=64, causal=True, fused=False),
        # the attention of the benchmark's transformer block: batch 32, 512 rows, 32 heads of 128
        dict(name="prompt block", op="prompt", dtype="bf16", seqs=32, shortest=512, longest=512, prefix=0, mix=2,
             q_heads=32, kv_heads=32, head_dim=128, causal=False, fused=False),
        # a server's mixed batch of prompts, one token to some thousand, q, k and v slices of one projection
        dict(name="prompt packed", op="prompt", dtype="bf16", seqs=24, shortest=1, longest=2111, prefix=0, mix=3,
             q_heads=32, kv_heads=8, head_dim=128, causal=True, fused=True),
        # one long document
        dict(name="prompt long", op="prompt", dtype="bf16", seqs=1, shortest=8192, longest=8192, prefix=0, mix=4,
             q_heads=32, kv_heads=8, head_dim=128, causal=True, fused=False),
        # one user, a short context: latency counts
        dict(name="decode one user", op="decode", dtype="bf16", seqs=1, shortest=333, longest=333, mix=5,
             q_heads=8, kv_heads=2, head_dim=64, page=16),
        # a batch of 32 users of the benchmark's block (32 heads, none shared), contexts from one token up
        dict(name="decode batch", op="decode", dtype="bf16", seqs=32, shortest=1, longest=1023, mix=6,
             q_heads=32, kv_heads=32, head_dim=128, page=16),
        # two users with long documents: few rows, a long axis to split
        dict(name="decode long", op="decode", dtype="f16", seqs=2, shortest=20011, longest=30001, mix=7,
             q_heads=32, kv_heads=8, head_dim=128, page=64),
        # a full server: many users with contexts of all lengths
        dict(name="decode server", op="decode", dtype="bf16", seqs=64, shortest=1500, longest=16384, mix=8,
             q_heads=32, kv_heads=8, head_dim=128, page=32),
        # the new token of each of 61 users
        dict(name="write step", op="write", dtype="bf16", seqs=61, shortest=1, longest=1, mix=9,
             kv_heads=8, head_dim=128, page=16, layers=2),
        # the keys and values of a batch of prompts
        dict(name="write prompts", op="write", dtype="bf16", seqs=24, shortest=7, longest=2111, mix=10,
             kv_heads=32, head_dim=128, page=16, layers=1),
        # a beam search's fork: 8 parents, 64 children, the last page of each copied in every layer
        dict(name="pages fork", op="fork", dtype="bf16", seqs=8, children=64, shortest=40, longest=700, mix=11,
             kv_heads=8, head_dim=128, page=16, layers=32, spare=96),
        # a pool with holes after sequences have ended, moved together
        dict(name="pages compact", op="compact", dtype="bf16", seqs=40, children=6, shortest=20, longest=900, mix=12,
             kv_heads=8, head_dim=128, page=16, layers=8, spare=700),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "decode", "decode", "write", "fork", "compact"])
    case = dict(op=op, dtype=rng.choice(["bf16", "f16"]), mix=rng.randrange(1 << 20), head_dim=rng.choice([64, 96, 128, 128]))
    kv = rng.choice([1, 2, 4, 8, 16])
    if op == "prompt":
        q_heads = kv * rng.choice([1, 2, 3, 4, 8]) if kv <= 4 else kv * rng.choice([1, 2])
        longest = _log(rng, 1, 6000)
        seqs = min(_log(rng, 1, 48), max(1, 16384 // longest), max(1, 500000000 // (longest * longest * q_heads)))
        case.update(seqs=seqs, shortest=rng.choice([1, longest, _log(rng, 1, longest)]), longest=longest,
                    prefix=rng.choice([0, 0, _log(rng, 1, 700)]), q_heads=q_heads, kv_heads=kv,
                    causal=rng.random() < 0.75, fused=False)
        case["fused"] = case["prefix"] == 0 and rng.random() < 0.5
    elif op == "decode":
        longest = _log(rng, 1, 32768)
        seqs = min(_log(rng, 1, 200), max(1, 3200000 // (longest * kv)))
        case.update(seqs=seqs, shortest=rng.choice([0, 1, longest, _log(rng, 1, longest)]), longest=longest,
                    q_heads=kv * rng.choice([1, 2, 3, 4, 7, 8, 16]), kv_heads=kv, page=rng.choice([8, 16, 24, 32, 64, 128]))
    elif op == "write":
        longest = _log(rng, 1, 4096)
        seqs = min(_log(rng, 1, 256), max(1, 32768 // longest))
        case.update(seqs=seqs, shortest=rng.choice([0, 1, longest]), longest=longest, kv_heads=kv,
                    page=rng.choice([8, 16, 24, 32, 64, 128]), layers=rng.choice([1, 2, 3]))
    else:
        longest = _log(rng, 1, 900)
        case.update(seqs=_log(rng, 1, 40), children=_log(rng, 1, 64), shortest=rng.choice([1, longest]), longest=longest,
                    kv_heads=min(kv, 8), page=rng.choice([8, 16, 24, 32, 64]), layers=_log(rng, 1, 8), spare=_log(rng, 70, 700))
    return case


# ---------------------------------------------------------------------------
# What a case's numbers stand for: lengths, pages and reference counts, from the case alone
# ---------------------------------------------------------------------------

def _lengths(case):
    """One length a sequence, spread over the logarithm; the last one is the longest."""
    r = random.Random(case["mix"])
    lo, hi = max(1, case["shortest"]), case["longest"]
    lens = [_log(r, lo, hi) for _ in range(case["seqs"] - 1)] + [hi]
    if case["shortest"] == 0 and case["seqs"] > 1:
        lens[0] = 0
    return lens


def _pages(case):
    """Lengths, page table and reference counts of a cache that has been in use: pages in no order, holes between."""
    r = random.Random(case["mix"] + 1)
    page = case["page"]
    lens = _lengths(case)
    if case["op"] == "write":  # the tokens to write follow a context already there
        lens = [n + r.randrange(0, 200) for n in lens]
    need = [-(-n // page) for n in lens]
    pages = sum(need) + case.get("spare", max(4, sum(need) // 8))
    order = r.sample(range(pages), sum(need))
    table, refs, at = [], [0] * pages, 0
    for n in need:
        table.append(order[at:at + n])
        at += n
        for p in table[-1]:
            refs[p] = 1
    if case["op"] == "compact":  # some sequences share whole pages with a fork of them
        for i in range(min(case["children"], case["seqs"])):
            whole = lens[i] // page
            table.append(table[i][:whole])
            lens.append(whole * page)
            for p in table[-1]:
                refs[p] += 1
    if case["op"] == "fork":
        table += [[] for _ in range(case["children"])]
        lens += [0] * case["children"]
    return lens, table, refs


def _parents(case):
    r = random.Random(case["mix"] + 2)
    return [r.randrange(case["seqs"]) for _ in range(case["children"])]


def work(case):
    d = case["head_dim"]
    if case["op"] == "prompt":
        lens, pre = _lengths(case), case["prefix"]
        rows, keys = sum(lens), sum(n + pre for n in lens)
        pairs = sum(n * pre + n * (n + 1) // 2 if case["causal"] else n * (n + pre) for n in lens)
        return {"bytes": 2 * d * (2 * rows * case["q_heads"] + 2 * keys * case["kv_heads"]) + 4 * rows * case["q_heads"],
                "flops": 4 * d * case["q_heads"] * pairs}
    if case["op"] == "decode":
        lens, table, _ = _pages(case)
        return {"bytes": 2 * d * (2 * sum(lens) * case["kv_heads"] + 2 * len(lens) * case["q_heads"])
                + 4 * (len(lens) * (2 + case["q_heads"]) + sum(len(t) for t in table)),
                "flops": 4 * d * case["q_heads"] * sum(lens)}
    row = 2 * 2 * d * case["kv_heads"]  # one token's key and value
    if case["op"] == "write":
        lens, _, _ = _pages(case)
        return {"bytes": 2 * row * sum(_lengths(case)) + 12 * len(lens), "flops": 0}
    lens, table, refs = _pages(case)
    if case["op"] == "fork":
        rows = sum(lens[p] % case["page"] for p in _parents(case))
        return {"bytes": 2 * row * rows * case["layers"] + 8 * sum(len(table[p]) for p in _parents(case)) + 4 * len(refs), "flops": 0}
    live = sum(1 for n in refs if n)
    moved = sum(1 for n in refs[live:] if n)
    return {"bytes": 2 * row * case["page"] * moved * case["layers"] + 8 * len(refs) + 8 * sum(map(len, table)), "flops": 0}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

_contexts = []


def _context():
    from tosa_b200 import _lib
    if not _contexts:
        _contexts.append(_lib.Context(torch.cuda.current_device()))
    return _contexts[0]


def _normal(g, shape, dtype, std=1.0):
    x = torch.empty(shape, dtype=dtype, device="cuda")
    return x.normal_(0.0, std, generator=g)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _offsets(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return _ints(at)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt, d = DTYPES[case["dtype"]], case["head_dim"]
    s = dict(case=case, scale=1.0 / math.sqrt(d))
    if case["op"] == "prompt":
        lens, pre, hq, hk = _lengths(case), case["prefix"], case["q_heads"], case["kv_heads"]
        keys = [n + pre for n in lens]
        if case["fused"]:  # one projection's rows: q, k and v heads side by side
            qkv = _normal(g, (sum(lens), hq + 2 * hk, d), dt)
            s.update(q=qkv[:, :hq], k=qkv[:, hq:hq + hk], v=qkv[:, hq + hk:])
        else:
            s.update(q=_normal(g, (sum(lens), hq, d), dt), k=_normal(g, (sum(keys), hk, d), dt),
                     v=_normal(g, (sum(keys), hk, d), dt))
        s.update(cu_q=_offsets(lens), cu_k=_offsets(keys), max_q=max(lens), max_k=max(keys))
        if own:
            s["ctx"] = _context()
        return s
    lens, table, refs = _pages(case)
    width = max(1, max(len(t) for t in table))
    shape = (case.get("layers", 1), len(refs), case["kv_heads"], case["page"], d)
    s.update(k_pages=_normal(g, shape, dt), v_pages=_normal(g, shape, dt), lengths=_ints(lens), refs=_ints(refs),
             page_table=_ints([t + [-1] * (width - len(t)) for t in table]), longest=max(lens))
    if case["op"] == "decode":
        # the server's order of its sequences is not the cache's
        slots = list(range(len(lens)))
        random.Random(case["mix"] + 3).shuffle(slots)
        s.update(slots=_ints(slots), q=_normal(g, (len(lens), case["q_heads"], d), dt))
    elif case["op"] == "write":
        new = _lengths(case)
        s.update(slots=_ints(list(range(len(lens)))), offsets=_offsets(new), tokens=sum(new),
                 k=_normal(g, (sum(new), case["kv_heads"], d), dt), v=_normal(g, (sum(new), case["kv_heads"], d), dt))
    elif case["op"] == "fork":
        s.update(parents=_ints(_parents(case)), children=_ints([case["seqs"] + i for i in range(case["children"])]))
    else:
        s.update(page_table_out=torch.empty_like(s["page_table"]), refs_out=torch.empty_like(s["refs"]))
    if own:
        from tosa_b200.attention import PagedCache
        s["cache"] = PagedCache(_context(), s["k_pages"], s["v_pages"], s["page_table"], s["lengths"], s["refs"])
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def run(s):
    op = s["case"]["op"]
    if own:
        return {"prompt": _own_prompt, "decode": _own_decode, "write": _own_write, "fork": _own_fork,
                "compact": _own_compact}[op](s)
    return {"prompt": _prompt, "decode": _decode, "write": _write, "fork": _fork, "compact": _compact}[op](s)


def _own_prompt(s):
    from tosa_b200.attention import attention
    out, lse = attention(s["ctx"], s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], causal=s["case"]["causal"], scale=s["scale"])
    return {"out": out, "lse": lse}


def _own_decode(s):
    out, lse = s["cache"].attend(0, s["slots"], s["q"], scale=s["scale"])
    return {"out": out, "lse": lse}


def _own_write(s):
    s["cache"].write(s["case"]["layers"] - 1, s["slots"], s["offsets"], s["k"], s["v"])
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _own_fork(s):
    s["cache"].fork(s["parents"], s["children"])
    return _cache_state(s, s["page_table"], s["refs"])


def _own_compact(s):
    s["cache"].compact(s["page_table_out"], s["refs_out"])
    return _cache_state(s, s["page_table_out"], s["refs_out"])


def _cache_state(s, table, refs):
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"], "page_table": table, "refs": refs, "lengths": s["lengths"]}


def _softmax_product(scores, mask, v):
    """softmax over the last axis where `mask` holds, times v; and the logarithm of the sum of exponentials."""
    scores = torch.where(mask, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    out = (p @ v) / torch.where(total == 0, 1.0, total)
    return out, (top + torch.log(total)).squeeze(-1)


def _prompt(s):
    q, k, v, cu_q, cu_k = s["q"], s["k"], s["v"], s["cu_q"].long(), s["cu_k"].long()
    n, mq, mk = cu_q.numel() - 1, s["max_q"], s["max_k"]
    hq, hk, d = q.shape[1], k.shape[1], q.shape[2]
    lq, lk = cu_q.diff()[:, None], cu_k.diff()[:, None]
    iq, ik = torch.arange(mq, device=q.device)[None], torch.arange(mk, device=q.device)[None]
    in_q, in_k = iq < lq, ik < lk
    rows = torch.where(in_q, cu_q[:-1, None] + iq, 0)
    keys = torch.where(in_k, cu_k[:-1, None] + ik, 0)
    qp = q[rows].float().reshape(n, mq, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(n, hk, hq // hk * mq, d)
    kp, vp = k[keys].float().permute(0, 2, 3, 1), v[keys].float().permute(0, 2, 1, 3)
    mask = in_k[:, None, :].expand(n, mq, mk)
    if s["case"]["causal"]:
        mask = mask & (ik[:, None, :] <= (iq + lk - lq)[:, :, None])
    mask = mask[:, None, None].expand(n, 1, hq // hk, mq, mk).reshape(n, 1, -1, mk)
    out, lse = _softmax_product((qp @ kp) * s["scale"], mask, vp)
    out = out.reshape(n, hk, hq // hk, mq, d).permute(0, 3, 1, 2, 4).reshape(n, mq, hq, d)
    lse = lse.reshape(n, hq, mq).permute(0, 2, 1)
    return {"out": out[in_q].to(q.dtype), "lse": lse[in_q].T.contiguous()}


def _decode(s):
    q, slots, page, d = s["q"], s["slots"].long(), s["case"]["page"], s["case"]["head_dim"]
    n, hk = q.shape[0], s["case"]["kv_heads"]
    width = max(1, -(-s["longest"] // page))
    table = s["page_table"][slots, :width].clamp(min=0).long()
    lens = s["lengths"][slots]
    k = s["k_pages"][0][table].float().transpose(1, 2).reshape(n, hk, width * page, d)
    v = s["v_pages"][0][table].float().transpose(1, 2).reshape(n, hk, width * page, d)
    mask = (torch.arange(width * page, device=q.device) < lens[:, None])[:, None, None]
    out, lse = _softmax_product((q.float().reshape(n, hk, -1, d) @ k.transpose(2, 3)) * s["scale"], mask, v)
    return {"out": out.reshape(n, -1, d).to(q.dtype), "lse": lse.reshape(n, -1)}


def _write(s):
    page, layer = s["case"]["page"], s["case"]["layers"] - 1
    offsets, slots = s["offsets"].long(), s["slots"].long()
    token = torch.arange(s["tokens"], device=offsets.device)
    i = torch.searchsorted(offsets, token, right=True) - 1
    at = s["lengths"].long()[slots[i]] - (offsets[i + 1] - token)
    p = s["page_table"].long()[slots[i], at // page]
    s["k_pages"][layer][p, :, at % page] = s["k"]
    s["v_pages"][layer][p, :, at % page] = s["v"]
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _fork(s):
    page, table, lengths, refs = s["case"]["page"], s["page_table"], s["lengths"], s["refs"]
    parents, children = s["parents"].long(), s["children"].long()
    # the children's former pages go back
    old = table[children].long()
    refs.scatter_add_(0, old.clamp(min=0).reshape(-1), -(old >= 0).int().reshape(-1))
    # whole pages are shared
    n = lengths[parents]
    whole, rest = (n // page).long(), n % page
    shared = torch.arange(table.shape[1], device=table.device) < whole[:, None]
    new = torch.where(shared, table[parents], -1)
    refs.scatter_add_(0, new.clamp(min=0).long().reshape(-1), shared.int().reshape(-1))
    # a page that is partly filled is copied to the lowest free page
    part = torch.nonzero(rest)[:, 0]
    free = torch.nonzero(refs == 0)[:, 0][:part.numel()]
    src = table[parents[part], whole[part]].long()
    new[part, whole[part]] = free.int()
    refs[free] = 1
    filled = (torch.arange(page, device=table.device) < rest[part][:, None])[None, :, None, :, None]
    for pages in (s["k_pages"], s["v_pages"]):
        pages[:, free] = torch.where(filled, pages[:, src], pages[:, free])
    table[children] = new
    lengths[children] = n
    return _cache_state(s, table, refs)


def _compact(s):
    table, refs = s["page_table"], s["refs"]
    live = refs > 0
    count, index = live.sum(), torch.arange(refs.numel(), device=refs.device)
    src = torch.nonzero(live & (index >= count))[:, 0]
    dst = torch.nonzero(~live & (index < count))[:, 0]
    to = index.clone()
    to[src] = dst
    refs_out = refs.clone()
    refs_out[dst] = refs[src]
    refs_out[src] = 0
    table_out = torch.where(table >= 0, to[table.clamp(min=0).long()].int(), -1)
    for pages in (s["k_pages"], s["v_pages"]):
        pages[:, dst] = pages[:, src]
    return _cache_state(s, table_out, refs_out)


# ---------------------------------------------------------------------------
# The definition in 64 bits, one sequence at a time
# ---------------------------------------------------------------------------

def _exact_rows(q, k, v, limits, scale):
    """q [h, r, d], k and v [n, d] in 64 bits; row i sees the keys before limits[i]."""
    out = torch.zeros_like(q)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    if k.shape[0] and q.shape[1]:
        scores = torch.einsum("hrd,nd->hrn", q, k) * scale
        hidden = torch.arange(k.shape[0], device=q.device)[None, :] >= limits[:, None]
        scores.masked_fill_(hidden[None], -math.inf)
        lse = torch.logsumexp(scores, -1)
        weights = torch.exp(scores - torch.where(lse == -math.inf, 0.0, lse)[..., None])
        out = torch.einsum("hrn,nd->hrd", weights, v)
    return out, lse


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    scale, op = s["scale"], case["op"]
    if op == "prompt":
        hq, hk = case["q_heads"], case["kv_heads"]
        g = hq // hk
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        lse = torch.zeros((hq, s["q"].shape[0]), dtype=torch.float64, device="cuda")
        cq, ck = s["cu_q"].tolist(), s["cu_k"].tolist()
        for b in range(len(cq) - 1):
            lq, lk = cq[b + 1] - cq[b], ck[b + 1] - ck[b]
            for h in range(hk):
                k, v = (s[x][ck[b]:ck[b + 1], h].double() for x in "kv")
                for r0 in range(0, lq, 2048):
                    r1 = min(lq, r0 + 2048)
                    at = torch.arange(r0, r1, device="cuda")
                    limits = at + (lk - lq) + 1 if case["causal"] else torch.full_like(at, lk)
                    q = s["q"][cq[b] + r0:cq[b] + r1, h * g:(h + 1) * g].double().transpose(0, 1)
                    o, l = _exact_rows(q, k, v, limits, scale)
                    out[cq[b] + r0:cq[b] + r1, h * g:(h + 1) * g] = o.transpose(0, 1)
                    lse[h * g:(h + 1) * g, cq[b] + r0:cq[b] + r1] = l
        return {"out": out, "lse": lse}
    if op == "decode":
        hk, g, page = case["kv_heads"], case["q_heads"] // case["kv_heads"], case["page"]
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device="cuda")
        table, lens = s["page_table"].tolist(), s["lengths"].tolist()
        for i, slot in enumerate(s["slots"].tolist()):
            n = lens[slot]
            pages = torch.tensor(table[slot][:-(-n // page)], dtype=torch.int64, device="cuda")
            for h in range(hk):
                k, v = (s[x][0, pages, h].double().reshape(-1, case["head_dim"])[:n] for x in ("k_pages", "v_pages"))
                q = s["q"][i, h * g:(h + 1) * g].double()[:, None]
                o, l = _exact_rows(q, k, v, torch.tensor([n], device="cuda"), scale)
                out[i, h * g:(h + 1) * g], lse[i, h * g:(h + 1) * g] = o[:, 0], l[:, 0]
        return {"out": out, "lse": lse}
    page, table, lens, refs = case["page"], s["page_table"].tolist(), s["lengths"].tolist(), s["refs"].tolist()
    kp, vp = s["k_pages"], s["v_pages"]
    if op == "write":
        at = s["offsets"].tolist()
        for i, slot in enumerate(s["slots"].tolist()):
            n, t = at[i + 1] - at[i], at[i]
            while n:  # as far as the page goes
                pos = lens[slot] - n
                c = min(n, page - pos % page)
                for pages, new in ((kp, s["k"]), (vp, s["v"])):
                    pages[-1, table[slot][pos // page], :, pos % page:pos % page + c] = new[t:t + c].transpose(0, 1)
                n, t = n - c, t + c
        return {"k_pages": kp.double(), "v_pages": vp.double()}
    if op == "fork":
        for parent, child in zip(s["parents"].tolist(), s["children"].tolist()):
            lens[child] = lens[parent]
            for j in range(lens[parent] // page):
                table[child][j] = table[parent][j]
                refs[table[parent][j]] += 1
        for parent, child in zip(s["parents"].tolist(), s["children"].tolist()):
            j, rest = divmod(lens[parent], page)
            if rest:
                to = refs.index(0)
                refs[to], table[child][j] = 1, to
                for pages in (kp, vp):
                    pages[:, to, :, :rest] = pages[:, table[parent][j], :, :rest]
    else:
        while True:
            live = [p for p, n in enumerate(refs) if n]
            src = next((p for p in live if p >= len(live)), None)
            if src is None:
                break
            to = refs.index(0)
            refs[to], refs[src] = refs[src], 0
            table = [[to if p == src else p for p in row] for row in table]
            kp[:, to], vp[:, to] = kp[:, src], vp[:, src]
    return {"k_pages": kp.double(), "v_pages": vp.double(), "page_table": _ints(table), "refs": _ints(refs), "lengths": _ints(lens)}
