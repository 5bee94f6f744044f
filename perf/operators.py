"""What the paged key-value cache's operators are measured on: their cases, inputs, plain forms and exact values.

Three operators of a server that keeps the keys and values of many sequences in one pool of fixed-size pages:

  tables     the pages of the sequences that grow are taken from the free list, and every new token gets its slot and position; a
             truncation gives the pages back (reserve + truncate)
  append     queries and keys are rotated, keys and values go to their tokens' slots, in bf16 or e4m3
  attention  the new tokens' queries over their sequences' pages: one token, a few drafted ones, a video frame's, a prompt's

The head layouts are those of this repository's language models: 28 query / 4 key-value heads of 128 channels (the 7B model), 8 / 2 of 64
and 4 / 2 of 64 (the small ones), 7 / 1 of 128.  A frame is 36 or 49 tokens, a ring cache 2,048 keys, the longest measured growing
cache 21,655 keys, the position table 32,768 rows, a server steps 16 streams at once.
"""
import math

import numpy as np
import torch

own = False                      # False: the plain form; True: the framework's kernels

POSITIONS = 32768                # rows of the position table
THETA = 1e6
E4M3_MAX = 448.0
HEADS = ((28, 4, 128), (28, 4, 128), (8, 2, 64), (4, 2, 64), (7, 1, 128))     # drawn from; the 7B layout twice as often


def listed():
    return [
        # sixteen live streams each about to generate one token: the smallest call, latency alone
        dict(name="tables_tokens", op="tables", requests=16, count=1, longest=21655, page=64),
        # a batch of questions of up to 512 tokens admitted at once: 65,000 tokens get their slots
        dict(name="tables_prompts", op="tables", requests=256, count=512, longest=4096, page=32),
        # one generated token for each of sixteen streams
        dict(name="append_tokens", op="append", requests=16, count=1, heads=28, kv_heads=4, dim=128, page=64, kind="bf16"),
        # one frame of 36 tokens for each of eight streams into an 8-bit cache
        dict(name="append_frames_e4m3", op="append", requests=8, count=36, heads=28, kv_heads=4, dim=128, page=64, kind="e4m3"),
        # prompts of ragged lengths, 16,000 tokens in all
        dict(name="append_prompts", op="append", requests=16, count=2048, heads=28, kv_heads=4, dim=128, page=64, kind="bf16"),
        # a response to one stream: one token over a ring's worth of keys
        dict(name="token_one", op="attention", requests=1, tokens=1, longest=2048, heads=28, kv_heads=4, dim=128, page=64, kind="bf16", window=0),
        # responses to sixteen streams of ragged lengths, up to ten minutes of video each
        dict(name="token_streams", op="attention", requests=16, tokens=1, longest=21655, heads=28, kv_heads=4, dim=128, page=64, kind="bf16", window=0),
        # sixty-four conversations over an 8-bit cache
        dict(name="token_many_e4m3", op="attention", requests=64, tokens=1, longest=16384, heads=28, kv_heads=4, dim=128, page=32, kind="e4m3", window=0),
        # the small model with a sliding window over long sequences, few keys to a page
        dict(name="token_window", op="attention", requests=32, tokens=1, longest=32768, heads=8, kv_heads=2, dim=64, page=16, kind="bf16", window=2048),
        # drafted tokens checked at once, up to eight a stream
        dict(name="drafts_e4m3", op="attention", requests=16, tokens=8, longest=8192, heads=28, kv_heads=4, dim=128, page=64, kind="e4m3", window=0),
        # one frame of each of eight growing streams
        dict(name="frames", op="attention", requests=8, tokens=36, longest=21655, heads=28, kv_heads=4, dim=128, page=64, kind="bf16", window=0),
        # two long questions behind their videos, the matrix product's share of the work at its largest
        dict(name="prompts", op="attention", requests=2, tokens=4096, longest=8192, heads=28, kv_heads=4, dim=128, page=64, kind="bf16", window=0),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], evenly over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("tables", "append", "attention", "attention"))
    page = rng.choice((16, 32, 64, 128))
    if op == "tables":
        requests = _spread(rng, 1, 256)
        return dict(op=op, requests=requests, count=_spread(rng, 1, 131072 // requests if requests > 64 else 2048), longest=_spread(rng, 64, 30000), page=page)
    heads, kv_heads, dim = rng.choice(HEADS)
    kind = rng.choice(("bf16", "bf16", "e4m3"))
    if op == "append":
        requests = _spread(rng, 1, 64)
        return dict(op=op, requests=requests, count=_spread(rng, 1, 30000 // requests), heads=heads, kv_heads=kv_heads, dim=dim, page=page, kind=kind)
    requests = _spread(rng, 1, 64)
    longest = _spread(rng, 64, min(32768, (1 << 20) // requests))
    most = min(longest, 4096, max(1, (1 << 25) // (requests * longest)))
    tokens = rng.choice((1, min(most, rng.randint(2, 8)), _spread(rng, 1, most)))
    return dict(op=op, requests=requests, tokens=tokens, longest=longest, heads=heads, kv_heads=kv_heads, dim=dim, page=page, kind=kind,
                window=rng.choice((0, 0, 0, _spread(rng, 16, longest))))


# ---- inputs -------------------------------------------------------------------------------------------------------------------------

def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _ragged(rs, n, low, high):
    """n whole numbers of [low, high], the highest among them."""
    x = rs.randint(low, high + 1, n)
    x[rs.randint(n)] = high
    return x.astype(np.int64)


def _pool(rs, lens, tables, page, pages):
    """Block tables of `tables` sequences of these lengths over a pool of `pages` pages in a random order, and the free list behind them."""
    blocks = -(-lens // page)
    wide = max(1, -(-POSITIONS // page))
    total = int(blocks.sum())
    order = rs.permutation(pages).astype(np.int32)
    table = np.full((tables, wide), -1, np.int32)
    row = np.repeat(np.arange(tables), blocks)
    at = np.arange(total) - np.repeat(np.cumsum(blocks) - blocks, blocks)
    table[row, at] = order[:total]
    free = np.zeros(pages, np.int32)
    free[:pages - total] = order[total:]
    return table, free


def _pages(gen, dev, pages, kv_heads, page, dim, kind):
    x = torch.empty((1, pages, kv_heads, page, dim), dtype=torch.bfloat16, device=dev).normal_(generator=gen)
    return x if kind == "bf16" else (x * 60).clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)


def _case_numbers(case, rs):
    """Lengths and counts of a case: (sequences in the tables, which of them take part, their lengths, their new tokens).  How many tokens
    there are is the case's, who has how many the seed's."""
    n = case["requests"]
    tables = n + n // 8 + 1
    seqs = rs.permutation(tables)[:n]
    most = case["tokens" if case["op"] == "attention" else "count"]
    low = {"attention": most if most in (36, 49) else max(1, most // 2), "append": most if most <= 49 else most // 8, "tables": 1 if most == 1 else 0}[case["op"]]
    counts = rs.permutation(_ragged(np.random.RandomState(n * 65537 + most), n, low, most))
    if case["op"] == "attention":
        lens = _ragged(rs, tables, max(1, case["longest"] // 8), case["longest"])
        lens[seqs[0]] = case["longest"]
        lens[seqs] = np.maximum(lens[seqs], counts)
    elif case["op"] == "append":
        lens = _ragged(rs, tables, 0, POSITIONS - most) if most <= 512 else np.zeros(tables, np.int64)
        lens[seqs] += counts
    else:
        lens = _ragged(rs, tables, 0, case["longest"])
    return tables, seqs, lens, counts


def prepare(case, seed):
    dev = _device()
    rs = np.random.RandomState(seed % (1 << 32))
    gen = torch.Generator(device=dev).manual_seed(seed)
    tables, seqs, lens, counts = _case_numbers(case, rs)
    n, total, page = len(seqs), int(counts.sum()), case["page"]
    s = {"op": case["op"], "page": page, "tokens": total, "most": int(counts.max()), "longest": int(lens[seqs].max())}
    if case["op"] == "append":
        # the pool of a server that holds just these tokens' pages: what the call writes lies anywhere in it
        first = lens[seqs] - counts
        stored = np.zeros(tables, np.int64)
        stored[seqs] = counts + first % page
        pages = int((-(-counts // page) + 1).sum()) + 8
        table, free = _pool(rs, stored, tables, page, pages)
        req = np.repeat(np.arange(n), counts)
        within = np.arange(total) - np.repeat(np.cumsum(counts) - counts, counts)
        off = (first % page)[req] + within
        s["slots"] = torch.from_numpy(table[seqs[req], off // page] * page + (off % page).astype(np.int32)).to(dev)
        s["positions"] = torch.from_numpy((first[req] + within).astype(np.int32)).to(dev)
    else:
        pages = tables * -(-(case["longest"] + (case["count"] if case["op"] == "tables" else 0)) // page)
        table, free = _pool(rs, lens, tables, page, pages)
        if case["op"] == "tables":
            s["need"] = int((-(-(lens[seqs] + counts) // page) - -(-lens[seqs] // page)).sum())
    put = lambda x: torch.from_numpy(np.ascontiguousarray(x).astype(np.int32)).to(dev)      # noqa: E731
    s.update(seqs=put(seqs), counts=put(counts), lens=put(lens), kept=put(lens[seqs]), table=put(table), free=put(free), n_free=put([len(free) - int((table >= 0).sum())]),
             cu=put(np.concatenate([[0], np.cumsum(counts)])))
    hq, hk, dim, kind = (case.get(k) for k in ("heads", "kv_heads", "dim", "kind"))
    if case["op"] != "tables":
        s.update(heads=hq, kv_heads=hk, dim=dim, kind=kind, window=case.get("window", 0))
        s["k_pages"], s["v_pages"] = (_pages(gen, dev, pages, hk, page, dim, kind) for _ in range(2))
        scale = torch.rand((2, 1, hk), generator=gen, device=dev) * 0.4 + 0.8
        s["k_scale"], s["v_scale"] = scale / 60 if kind == "e4m3" else torch.ones_like(scale)
    if case["op"] == "append":
        # what the fused projection writes: q | k | v of a token in one row
        s["qkv"] = torch.randn((total, (hq + 2 * hk) * dim), generator=gen, device=dev).mul_(1.5).bfloat16()
        inv = THETA ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=dev) / dim)
        angle = torch.arange(POSITIONS, dtype=torch.float64, device=dev)[:, None] * inv
        s["cos"], s["sin"] = (torch.cat((t, t), -1).bfloat16() for t in (angle.cos(), angle.sin()))
    if case["op"] == "attention":
        s["q"] = torch.randn((total, hq, dim), generator=gen, device=dev).mul_(1.5).bfloat16()
    if own:
        from aha_amd.paged import PagedKVCache
        more = {} if case["op"] == "tables" else dict(k_pages=s["k_pages"], v_pages=s["v_pages"])
        if kind == "e4m3":
            more.update(k_scale=s["k_scale"], v_scale=s["v_scale"])
        if case["op"] == "append":
            more["rope"] = (s["cos"], s["sin"])
        s["cache"] = PagedKVCache(pages, page, hk or 1, dim or 16, tables, table.shape[1], dtype=torch.float8_e4m3fn if kind == "e4m3" else torch.bfloat16,
                                  device=dev, block_table=s["table"], lens=s["lens"], free_pages=s["free"], n_free=s["n_free"], **more)
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------------------------

def run(state):
    if own:
        return {"tables": _own_tables, "append": _own_append, "attention": _own_attention}[state["op"]](state)
    return {"tables": _plain_tables, "append": _plain_append, "attention": _plain_attention}[state["op"]](state)


def _own_tables(s):
    c = s["cache"]
    slots, positions, cu, status = c.reserve(s["seqs"], s["counts"], s["tokens"])
    back = c.truncate(s["seqs"], s["kept"])
    return {"slots": slots, "positions": positions, "cu": cu, "status": status, "back": back, "table": c.block_table, "lens": c.lens, "free": c.free_pages, "n_free": c.n_free}


def _own_append(s):
    c, d = s["cache"], s["dim"]
    nq, nk = s["heads"] * d, s["kv_heads"] * d
    q, k, v = s["qkv"].split((nq, nk, nk), -1)
    return {"q": c.append(0, q, k, v, s["slots"], s["positions"]), "k": c.k_pages, "v": c.v_pages}


def _own_attention(s):
    return s["cache"].attention(0, s["q"], s["seqs"], s["cu"], max_q=s["most"], max_len=s["longest"], window=s["window"])


def _plain_tables(s):
    """Reserve: request i needs ceil((len + count) / page) - ceil(len / page) pages, taken from the end of the free list in the order of the
    requests; token t of it has position len + t and the slot page_of(position) * page + position % page.  Truncate: the same pages go back
    in the opposite order."""
    page, seqs, counts, table, lens, free, n_free = (s[k] for k in ("page", "seqs", "counts", "table", "lens", "free", "n_free"))
    seqs = seqs.long()
    before = lens[seqs].long()
    after = before + counts
    had, have = (before + page - 1) // page, (after + page - 1) // page
    need = have - had
    end = need.cumsum(0)
    cu = torch.zeros(len(seqs) + 1, dtype=torch.int32, device=seqs.device)
    cu[1:] = counts.cumsum(0)
    # every taken page: its request, and the place in the table it goes to
    p = torch.arange(s["need"], device=seqs.device)
    req = torch.searchsorted(end, p, right=True)
    at = seqs[req] * table.shape[1] + had[req] + p - (end - need)[req]
    source, flat = n_free - 1 - p, table.view(-1)
    flat[at] = free[source]
    lens[seqs] = after.int()
    n_free -= end[-1:].int()
    # the tokens
    t = torch.arange(s["tokens"], device=seqs.device)
    req = torch.searchsorted(cu[1:].long(), t, right=True)
    positions = before[req] + t - cu[req]
    slots = (table[seqs[req], positions // page] * page + positions % page).int()
    # truncated to what they were
    free[source] = flat[at]
    flat[at] = -1
    lens[seqs] = s["kept"]
    n_free += end[-1:].int()
    status = torch.zeros(2, dtype=torch.int32, device=seqs.device)
    return {"slots": slots, "positions": positions.int(), "cu": cu, "status": status, "back": status.clone(), "table": table, "lens": lens, "free": free, "n_free": n_free}


def _plain_append(s):
    """The pair (x[d], x[d + D/2]) turns by its position's angle; each value is rounded once, to its page's type."""
    n, d, page = s["tokens"], s["dim"], s["page"]
    q, k, v = (x.reshape(n, -1, d).float() for x in s["qkv"].split((s["heads"] * d, s["kv_heads"] * d, s["kv_heads"] * d), -1))
    at = s["positions"].long()
    cos, sin = s["cos"][at].float()[:, None], s["sin"][at].float()[:, None]
    turn = lambda x: x * cos + torch.cat((-x[..., d // 2:], x[..., :d // 2]), -1) * sin      # noqa: E731
    q, k = turn(q), turn(k)
    slot = s["slots"].long()
    for pages, x, scale in ((s["k_pages"], k, s["k_scale"]), (s["v_pages"], v, s["v_scale"])):
        if s["kind"] == "e4m3":
            x = (x / scale[0][:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8)
            pages[0].view(torch.uint8)[slot // page, :, slot % page] = x
        else:
            pages[0][slot // page, :, slot % page] = x.bfloat16()
    return {"q": q.bfloat16(), "k": s["k_pages"], "v": s["v_pages"]}


def _plain_attention(s):
    """softmax(q k^T / sqrt(D)) v over the keys at and before each query's position, no more than `window` of them; the last of a request's
    queries is at its sequence's last key.  All requests side by side, padded to the longest."""
    hq, hk, d, page = s["heads"], s["kv_heads"], s["dim"], s["page"]
    n, most = len(s["seqs"]), s["most"]
    cu, seqs = s["cu"].long(), s["seqs"].long()
    count, lens = cu[1:] - cu[:-1], s["lens"][seqs].long()
    blocks = -(-s["longest"] // page)
    at = s["table"][seqs, :blocks].long().clamp(min=0)

    def gather(pages, scale):
        x = pages[0].view(torch.uint8)[at].view(torch.float8_e4m3fn) if s["kind"] == "e4m3" else pages[0][at]
        x = x.float() * scale[0][:, None, None]
        return x.permute(0, 2, 1, 3, 4).reshape(n, hk, blocks * page, d)

    t = torch.arange(most, device=cu.device)
    token = (cu[:-1, None] + t).clamp(max=s["tokens"] - 1)
    q = s["q"][token].float().view(n, most, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(n, hk, -1, d)
    score = (q * d ** -0.5) @ gather(s["k_pages"], s["k_scale"]).transpose(-1, -2)
    position = (lens - count)[:, None] + t
    key = torch.arange(blocks * page, device=cu.device)
    seen = (key <= position[..., None]) & (key < lens[:, None, None]) & (position >= 0)[..., None]
    if s["window"]:
        seen &= key > position[..., None] - s["window"]
    score = score.view(n, hk, hq // hk, most, -1).masked_fill_(~seen[:, None, None], -math.inf)
    score -= score.amax(-1, keepdim=True).clamp(min=-1e30)
    p = score.exp_()
    out = (p.view(n, hk, -1, blocks * page) @ gather(s["v_pages"], s["v_scale"])).view(n, hk, hq // hk, most, d)
    out /= p.sum(-1, keepdim=True).clamp(min=1e-30)
    req = torch.searchsorted(cu[1:], torch.arange(s["tokens"], device=cu.device), right=True)
    within = torch.arange(s["tokens"], device=cu.device) - cu[req]
    return out.permute(0, 3, 1, 2, 4)[req, within].reshape(s["tokens"], hq, d).bfloat16()


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------------------

def work(case):
    rs = np.random.RandomState(1)
    _, seqs, lens, counts = _case_numbers(case, rs)
    lens, total = lens[seqs], int(counts.sum())
    if case["op"] == "tables":
        pages = int((-(-(lens + counts) // case["page"]) - -(-lens // case["page"])).sum())
        # counts, lengths in and out, kept lengths; each page from and to the free list and the table; a slot and a position a token
        return {"bytes": 4 * (len(seqs) * 6 + pages * 4 + total * 2), "flops": total}
    hq, hk, d, size = case["heads"], case["kv_heads"], case["dim"], 2 if case["kind"] == "bf16" else 1
    if case["op"] == "append":
        return {"bytes": total * (2 * hq * d * 2 + 2 * hk * d * (2 + size) + 8), "flops": total * (hq + hk) * d * 3}
    window = case["window"] or (1 << 30)
    first = np.maximum(0, lens - counts + 1 - window)                    # the first key that any of a request's queries sees
    at = np.concatenate([np.arange(n - c, n) for n, c in zip(lens, counts)])
    seen = np.minimum(at + 1, window)
    return {"bytes": int((lens - first).sum()) * 2 * hk * d * size + 2 * total * hq * d * 2, "flops": int(seen.sum()) * hq * d * 4}


# ---- the definition, in 64 bits ---------------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "tables":
        return None
    if case["op"] == "append":
        return _exact_append(s)
    return _exact_attention(s)


def _exact_append(s):
    d, half, page = s["dim"], s["dim"] // 2, s["page"]
    rows = s["qkv"].double().view(s["tokens"], -1, d)
    c, w = (s[x].double()[s["positions"].long()].unsqueeze(1) for x in ("cos", "sin"))
    out = torch.empty_like(rows)
    out[..., :half] = rows[..., :half] * c[..., :half] - rows[..., half:] * w[..., :half]
    out[..., half:] = rows[..., half:] * c[..., half:] + rows[..., :half] * w[..., half:]
    hq, hk = s["heads"], s["kv_heads"]
    answer = {"q": out[:, :hq].contiguous()}
    slot = s["slots"].long()
    for name, x in (("k", out[:, hq:hq + hk]), ("v", rows[:, hq + hk:])):
        pages = s[name + "_pages"].double()
        x = (x / s[name + "_scale"].double()[0][:, None])
        if s["kind"] == "e4m3":
            x = x.clamp(-E4M3_MAX, E4M3_MAX)
        flat = pages[0].transpose(1, 2).reshape(-1, hk, d).index_copy(0, slot, x.contiguous())     # [slot][head][channel]
        answer[name] = flat.view(-1, page, hk, d).transpose(1, 2).unsqueeze(0)
    return answer


def _exact_attention(s):
    hq, hk, d, page = s["heads"], s["kv_heads"], s["dim"], s["page"]
    out = torch.zeros((s["tokens"], hq, d), dtype=torch.float64, device=s["q"].device)
    cu, lens, seqs, table = (s[x].tolist() for x in ("cu", "lens", "seqs", "table"))
    for i, row in enumerate(seqs):
        n, first = lens[row], lens[row] - (cu[i + 1] - cu[i])
        pages = torch.tensor(table[row][:-(-n // page)], device=out.device)
        for h in range(hk):
            k, v = ((s[x + "_pages"][0][:, h].view(torch.uint8)[pages].view(s[x + "_pages"].dtype).double() * s[x + "_scale"][0][h].double()).reshape(-1, d)[:n] for x in "kv")
            heads = slice(h * hq // hk, (h + 1) * hq // hk)
            for a in range(cu[i], cu[i + 1], 512):
                b = min(a + 512, cu[i + 1])
                q = s["q"][a:b, heads].double()                          # [tokens][group][channel]
                logit = torch.einsum("tgd,kd->tgk", q, k) / math.sqrt(d)
                back = torch.arange(first + a - cu[i], first + b - cu[i], device=out.device)[:, None, None] - torch.arange(n, device=out.device)
                hidden = (back < 0) | (back >= s["window"]) if s["window"] else back < 0
                out[a:b, heads] = torch.softmax(logit.masked_fill(hidden, -math.inf), -1) @ v
    return out
