"""What the serving operators over a paged key / value cache cost: cases, inputs, plain forms and calls.

Three operators of a decoder's serving step, each with cases from the smallest
call to the largest:

  append  the rows of a fused q | k | v projection: RMS norm of each query and
          key head, position rotation, keys and values into a paged cache
          (bf16, or 4-bit codes with a scale and a minimum for each 64 values)
  attend  attention of the new rows over that cache (grouped heads, ragged
          lengths, one row or a few rows a sequence)
  sample  the next ids from the logits: temperature, top-k, top-p, min-p, and
          a race on given exponential random numbers

A page holds `page` tokens of every key / value head; the pool is uint8
[n_pages, kv_heads, block] with, in a block, the keys and then the values of
its tokens: bf16 [page][head_dim] each, or 4-bit codes [page][head_dim / 2]
(the even dimension in the low half of a byte) followed by bf16 (scale,
minimum) pairs [page][head_dim / 64][2].  A code c stands for minimum + c *
scale.  table [n_seq, max_pages] gives the page of each page slot of a
sequence.
"""
import math
import random

import torch

own = False

GROUP = 64       # dimensions that share a scale and a minimum
EPS = 1e-6
TABLE = 40960    # rows of the rotation tables

# (query heads, key / value heads, head dimension): the head layouts of the framework's decoders (12 and 25 heads of 64,
# 16 of 128), which keep their caches in fixed slots so far, and grouped ones as PagedDecoder's
HEADS = [(12, 12, 64), (25, 25, 64), (16, 16, 128), (32, 8, 128), (28, 4, 128), (64, 8, 128), (8, 1, 128), (16, 2, 256)]


def listed():
    return [
        # one sequence of the 12-head decoder appends its next token
        dict(name="append_1_h64", op="append", n_seq=1, rows=1, ctx=1024, heads=12, kv=12, hd=64, page=16, bits=16,
             f32=True, norm=False, rot=64, pairs=False),
        # a decode step of 32 sequences, projection in f32, 4-bit pages
        dict(name="append_32_q4", op="append", n_seq=32, rows=32, ctx=8192, heads=32, kv=8, hd=128, page=16, bits=4,
             f32=True, norm=True, rot=128, pairs=False),
        # the prompts of 5 requests in one pass, ragged, 4-bit pages, half of each head rotated in neighbouring pairs
        dict(name="append_4093_q4", op="append", n_seq=5, rows=4093, ctx=4096, heads=28, kv=4, hd=128, page=64, bits=4,
             f32=False, norm=True, rot=64, pairs=True),
        # the largest prompt pass, bf16 pages
        dict(name="append_16384", op="append", n_seq=16, rows=16384, ctx=2048, heads=16, kv=16, hd=128, page=32, bits=16,
             f32=False, norm=True, rot=128, pairs=False),
        # the start of a conversation: one short sequence
        dict(name="attend_1x37", op="attend", n_seq=1, new=1, ctx=37, heads=12, kv=12, hd=64, page=16, bits=16),
        # a decode step of 16 sequences of the 25-head decoder, lengths up to its 1024
        dict(name="attend_16x1024_h64", op="attend", n_seq=16, new=1, ctx=1024, heads=25, kv=25, hd=64, page=16, bits=16),
        # one long document, 4-bit pages
        dict(name="attend_1x32768_q4", op="attend", n_seq=1, new=1, ctx=32768, heads=32, kv=8, hd=128, page=32, bits=4),
        # verify rows of speculative decode: 4 new rows a sequence
        dict(name="attend_8x4096_q4_new4", op="attend", n_seq=8, new=4, ctx=4096, heads=64, kv=8, hd=128, page=64, bits=4),
        # the largest decode step: 64 sequences of 1 to 16384 tokens, 4-bit pages
        dict(name="attend_64x16384_q4", op="attend", n_seq=64, new=1, ctx=16384, heads=32, kv=8, hd=128, page=64, bits=4),
        # one request, top-k
        dict(name="sample_1_topk", op="sample", rows=1, vocab=50257, bf16=False, kind="topk", masked=False),
        # a decode batch whose requests each bring their own settings
        dict(name="sample_32_mixed", op="sample", rows=32, vocab=102400, bf16=False, kind="mixed", masked=True),
        # the largest batch: top-p and min-p over bf16 logits (many equal ones)
        dict(name="sample_256_topp", op="sample", rows=256, vocab=102400, bf16=True, kind="topp", masked=False),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def _size(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    op = rng.choice(["append", "attend", "sample"])
    most = max(_size(c) for c in listed() if c["op"] == op)
    while True:
        heads, kv, hd = rng.choice(HEADS)
        page, bits = rng.choice([16, 32, 64]), rng.choice([4, 16])
        if op == "append":
            rows = _log(rng, 1, 16384)
            n_seq = rows if rng.random() < 0.4 and rows <= 512 else min(rows, _log(rng, 1, 32))
            case = dict(op=op, n_seq=n_seq, rows=rows, ctx=_log(rng, 64, 16384), heads=heads, kv=kv, hd=hd, page=page,
                        bits=bits, f32=rng.random() < 0.5, norm=rng.random() < 0.7,
                        rot=rng.choice([0, hd // 2, hd, hd]), pairs=rng.random() < 0.4)
        elif op == "attend":
            case = dict(op=op, n_seq=_log(rng, 1, 128), new=rng.choice([1, 1, 1, 2, 4, 7, 16]), ctx=_log(rng, 16, 32768),
                        heads=heads, kv=kv, hd=hd, page=page, bits=bits)
        else:
            case = dict(op=op, rows=_log(rng, 1, 256), vocab=_log(rng, 1000, 131072), bf16=rng.random() < 0.5,
                        kind=rng.choice(["topk", "topp", "mixed", "none"]), masked=rng.random() < 0.3)
        if _size(case) <= most and 3072 not in case.values():  # a size that no configuration here has stays out
            return case


# ---- inputs -------------------------------------------------------------------


def _lengths(case):
    """Keys of each sequence after the new rows: 1 .. ctx, the last one ctx; the same for every seed."""
    r = random.Random(case["n_seq"] * 65537 + case["ctx"])
    n = [max(1, round(case["ctx"] * r.random())) for _ in range(case["n_seq"])]
    n[-1] = case["ctx"]
    return n


def _new_rows(case):
    """Rows of each sequence: one each, or ragged parts of all rows."""
    n, rows = case["n_seq"], case["rows"]
    cut = sorted(random.Random(rows * 8191 + n).sample(range(1, rows), n - 1))
    return [b - a for a, b in zip([0] + cut, cut + [rows])]


def _token_bytes(case):
    return 2 * case["hd"] if case["bits"] == 16 else case["hd"] // 2 + 4 * (case["hd"] // GROUP)


def _table(lengths, page, g, dev):
    """A shuffled pool: the page of each page slot (-1 past a sequence's end)."""
    need = [-(-n // page) for n in lengths]
    total, most = sum(need), max(need)
    ids = torch.randperm(total, generator=g, device=dev).to(torch.int32)
    slot = torch.arange(most, device=dev)[None]
    used = torch.tensor(need, device=dev)[:, None]
    first = torch.cumsum(used, 0) - used
    table = torch.where(slot < used, ids[(first + slot).clamp(max=total - 1)], torch.full((), -1, dtype=torch.int32, device=dev))
    return table.to(torch.int32).contiguous(), total


def _fill(case, pages, g, dev):
    """A pool of `pages` pages of keys and values as a decoder leaves them: a few strong key channels, values around zero."""
    kv, hd, page = case["kv"], case["hd"], case["page"]
    pool = torch.empty(pages, kv, 2 * page * _token_bytes(case), dtype=torch.uint8, device=dev)
    strong = 1 + 3 * (torch.rand(kv, 1, hd, generator=g, device=dev) < 0.04).float()
    step = max(1, (1 << 27) // (kv * page * hd))
    for a in range(0, pages, step):
        x = torch.randn(min(step, pages - a), kv, 2, page, hd, generator=g, device=dev)
        x[:, :, 0] *= strong
        pool[a:a + step] = _pack(x, case["bits"])
    return pool


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    s = dict(case=case, op=case["op"])
    if case["op"] == "sample":
        B, V, kind = case["rows"], case["vocab"], case["kind"]
        x = 2 * torch.randn(B, V, generator=g, device=dev)
        at = torch.randint(V, (B, 24), generator=g, device=dev)
        likely = 5 + 9 * torch.rand(B, 24, generator=g, device=dev)  # the few tokens that a model holds likely
        for a, v in zip(at.split(1, 1), likely.split(1, 1)):  # one after the other: an id that comes twice keeps its last value
            x.scatter_(1, a, v)
        if case["masked"]:
            x.masked_fill_(torch.rand(B, V, generator=g, device=dev) < 0.3, -math.inf)
        s["logits"] = x.to(torch.bfloat16) if case["bf16"] else x
        s["noise"] = torch.empty(B, V, device=dev).exponential_(generator=g)
        u = torch.rand(4, B, generator=g, device=dev)
        row = torch.arange(B, device=dev)
        s["temperature"], s["top_k"], s["top_p"], s["min_p"] = 0.6 + 0.7 * u[0], None, None, None
        if kind in ("topk", "mixed"):
            s["top_k"] = (20 + 80 * u[1]).to(torch.int32)
        if kind in ("topp", "mixed"):
            s["top_p"], s["min_p"] = 0.8 + 0.19 * u[2], 0.02 * u[3]
        if kind == "mixed":  # every fifth row greedy, others with one filter each, some with all, some with none
            s["temperature"] = torch.where(row % 5 == 4, 0.0, s["temperature"])
            s["top_k"] = torch.where(row % 4 == 1, 0, s["top_k"]).to(torch.int32)
            s["top_p"] = torch.where(row % 4 == 0, 1.0, s["top_p"])
            s["min_p"] = torch.where(row % 3 == 0, 0.0, s["min_p"])
        if own:
            from thvm_b200.sampling import Sampler
            s["sampler"] = Sampler(dev)
        return s
    H, kv, hd, page, bits = (case[k] for k in ("heads", "kv", "hd", "page", "bits"))
    if case["op"] == "append":
        new = _new_rows(case)
        r = random.Random(case["rows"] * 127 + case["ctx"])  # as many pages for every seed
        start = [r.randrange(case["ctx"]) if case["n_seq"] == case["rows"] else r.choice([0, r.randrange(case["ctx"])]) for _ in new]
        table, pages = _table([a + n for a, n in zip(start, new)], page, g, dev)
        n = torch.tensor(new, device=dev)
        s["seq"] = torch.arange(len(new), device=dev).repeat_interleave(n).to(torch.int32)
        first = (torch.cumsum(n, 0) - n)[s["seq"].long()]
        s["pos"] = (torch.tensor(start, device=dev)[s["seq"].long()] + torch.arange(case["rows"], device=dev) - first).to(torch.int32)
        x = torch.randn(case["rows"], (H + 2 * kv) * hd, generator=g, device=dev)
        s["qkv"] = x if case["f32"] else x.to(torch.bfloat16)
        if case["norm"]:
            s["g_q"], s["g_k"] = (1 + 0.2 * torch.randn(hd, generator=g, device=dev) for _ in range(2))
        if case["rot"]:
            f = 10000.0 ** (-torch.arange(case["rot"] // 2, device=dev, dtype=torch.float64) * 2 / case["rot"])
            a = torch.arange(TABLE, device=dev, dtype=torch.float64)[:, None] * f
            s["cos"], s["sin"] = a.cos().float(), a.sin().float()
        s["pool"] = _fill(case, pages, g, dev)
    else:
        lens = _lengths(case)
        table, pages = _table(lens, page, g, dev)
        s["pool"] = _fill(case, pages, g, dev)
        new = [min(case["new"], n) for n in lens]
        s["rows"] = new
        s["kv_len"] = torch.tensor(lens, dtype=torch.int32, device=dev)
        s["q_off"] = torch.tensor([0] + new, device=dev).cumsum(0).to(torch.int32) if case["new"] > 1 else None
        s["q"] = torch.randn(sum(new), H, hd, generator=g, device=dev).to(torch.bfloat16)
        s["scale"] = hd ** -0.5
    s["table"] = table
    if own:
        from thvm_b200.paged import PagedCache
        s["cache"] = PagedCache(s["pool"], table, page=page, head_dim=hd, bits=bits)
    return s


# ---- one pass -----------------------------------------------------------------


def run(state):
    return {"append": _append, "attend": _attend, "sample": _sample}[state["op"]](state)


def _append(s):
    case = s["case"]
    if own:
        q = s["cache"].append(s["qkv"], s["pos"], s["seq"], heads=case["heads"], g_q=s.get("g_q"), g_k=s.get("g_k"),
                              cos=s.get("cos"), sin=s.get("sin"), pairs=case["pairs"], eps=EPS)
        if case["bits"] == 16:
            return dict(q=q, pool=s["pool"].view(torch.bfloat16))
        k, v = s["cache"].read(s["pos"], s["seq"])
        return dict(q=q, k=k, v=v)
    H, kv, hd, page = case["heads"], case["kv"], case["hd"], case["page"]
    x = s["qkv"].float().view(-1, H + 2 * kv, hd)
    q, k, v = x[:, :H], x[:, H:H + kv], x[:, H + kv:]
    if case["norm"]:
        q, k = (t * torch.rsqrt((t * t).mean(-1, keepdim=True) + EPS) * w for t, w in ((q, s["g_q"]), (k, s["g_k"])))
    if case["rot"]:
        c, n = s["cos"][s["pos"].long()][:, None], s["sin"][s["pos"].long()][:, None]
        q, k = (_rotate(t, c, n, case["rot"], case["pairs"]) for t in (q, k))
    at = s["table"][s["seq"].long(), (s["pos"] // page).long()].long()
    row = (s["pos"] % page).long()
    both = torch.stack((k, v), 2)  # [rows, kv, 2, hd]
    if case["bits"] == 16:
        s["pool"].view(torch.bfloat16).view(-1, kv, 2, page, hd)[at, :, :, row] = both.to(torch.bfloat16)
        return dict(q=q.to(torch.bfloat16), pool=s["pool"].view(torch.bfloat16))
    codes, marks = _quantise(both)
    pool, half = s["pool"].view(-1, kv, 2, page * _token_bytes(case)), page * hd // 2
    pool[..., :half].view(-1, kv, 2, page, hd // 2)[at, :, :, row] = codes[..., 0::2] | codes[..., 1::2] << 4
    pool[..., half:].view(-1, kv, 2, page, 4 * (hd // GROUP))[at, :, :, row] = marks.reshape(*both.shape[:3], -1).view(torch.uint8)
    values = _values(pool[..., :half].view(-1, kv, 2, page, hd // 2)[at, :, :, row],
                     pool[..., half:].view(-1, kv, 2, page, 4 * (hd // GROUP))[at, :, :, row]).to(torch.bfloat16)
    return dict(q=q.to(torch.bfloat16), k=values[:, :, 0], v=values[:, :, 1])


def _rotate(t, c, n, rot, pairs):
    a, b = (t[..., 0:rot:2], t[..., 1:rot:2]) if pairs else (t[..., :rot // 2], t[..., rot // 2:rot])
    x, y = a * c - b * n, b * c + a * n
    turned = torch.stack((x, y), -1).flatten(-2) if pairs else torch.cat((x, y), -1)
    return torch.cat((turned, t[..., rot:]), -1)


def _quantise(x):
    """f32 [..., hd] to codes (uint8, one a value) and bf16 (scale, minimum) pairs [..., hd / 64, 2]."""
    y = x.unflatten(-1, (-1, GROUP))
    low = y.amin(-1, keepdim=True)
    scale = ((y.amax(-1, keepdim=True) - low) / 15).to(torch.bfloat16)
    low = low.to(torch.bfloat16)
    code = torch.where(scale > 0, torch.round((y - low.float()) / scale.float()), torch.zeros_like(y)).clamp(0, 15)
    return code.to(torch.uint8).flatten(-2), torch.cat((scale, low), -1)


def _values(codes, marks):
    """The values that packed codes [..., hd / 2] and their (scale, minimum) bytes stand for."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float().unflatten(-1, (-1, GROUP))
    m = marks.contiguous().view(torch.bfloat16).float().unflatten(-1, (-1, 2))
    return (m[..., 1:] + c * m[..., :1]).flatten(-2)


def _pack(x, bits):
    """Pages [n, kv, 2, page, hd] in the pool's bytes."""
    if bits == 16:
        return x.to(torch.bfloat16).flatten(2).view(torch.uint8)
    codes, marks = _quantise(x)
    packed = (codes[..., 0::2] | codes[..., 1::2] << 4).flatten(3)
    return torch.cat((packed, marks.flatten(3).view(torch.uint8)), -1).flatten(2)


def _keys_values(s):
    """Each sequence's keys and values in f32, [n_seq, 2, kv, slots * page, hd]."""
    case = s["case"]
    kv, hd, page = case["kv"], case["hd"], case["page"]
    x = s["pool"][s["table"].clamp(min=0).long()].unflatten(-1, (2, -1))  # [n_seq, slots, kv, 2, bytes]
    if case["bits"] == 16:
        x = x.view(torch.bfloat16).float().unflatten(-1, (page, hd))
    else:
        half = page * hd // 2
        x = _values(x[..., :half].unflatten(-1, (page, -1)), x[..., half:].unflatten(-1, (page, -1)))
    return x.permute(0, 3, 2, 1, 4, 5).flatten(3, 4)


def _attend(s):
    case = s["case"]
    if own:
        return s["cache"].attend(s["q"], s["kv_len"], q_off=s["q_off"], max_rows=case["new"], scale=s["scale"])
    H, kv, hd, n, R = case["heads"], case["kv"], case["hd"], case["n_seq"], case["new"]
    T = s["q"].shape[0]
    first = torch.arange(n, device=s["q"].device) if s["q_off"] is None else s["q_off"][:-1].long()
    count = torch.ones_like(first) if s["q_off"] is None else s["q_off"][1:].long() - first
    r = torch.arange(R, device=first.device)
    live = r < count[:, None]
    q = torch.where(live[..., None, None], s["q"].float()[(first[:, None] + r).clamp(max=T - 1)], 0.0)  # [n, R, H, hd]
    q = q.view(n, R, kv, H // kv, hd).permute(0, 2, 1, 3, 4).reshape(n, kv, -1, hd)
    x = _keys_values(s)
    z = (q @ x[:, 0].transpose(-1, -2)).view(n, kv, R, H // kv, -1) * s["scale"]
    last = s["kv_len"][:, None] - count[:, None] + r  # the key of the row itself
    hide = torch.arange(z.shape[-1], device=z.device) > last[..., None]
    z = z.masked_fill_(hide[:, None, :, None], -math.inf)
    p = (z - z.amax(-1, keepdim=True)).exp_()
    p /= p.sum(-1, keepdim=True)
    o = (p.flatten(2, 3) @ x[:, 1]).view(n, kv, R, H // kv, hd).permute(0, 2, 1, 3, 4).reshape(n, R, H, hd)
    return o.to(torch.bfloat16)[live]


def _sample(s):
    if own:
        tok, logp = s["sampler"](s["logits"], s["noise"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                                 min_p=s["min_p"])
        return dict(tok=tok, logp=logp)
    x, at = torch.sort(s["logits"].float(), dim=-1, descending=True, stable=True)
    V = x.shape[1]
    rank = torch.arange(V, device=x.device)
    t = s["temperature"][:, None]
    d = (x - x[:, :1]) / torch.where(t > 0, t, 1.0)
    keep = x > -math.inf
    if s["top_k"] is not None:
        k = s["top_k"][:, None]
        keep &= (k <= 0) | (rank < k)
    w = d.exp() * keep
    if s["top_p"] is not None:
        p = s["top_p"][:, None]
        before = w.cumsum(-1) - w
        keep &= (p >= 1) | (before < p * w.sum(-1, keepdim=True)) | (rank == 0)
    if s["min_p"] is not None:
        keep &= (d.exp() >= s["min_p"][:, None]) | (rank == 0)
    w = w * keep
    race = (d - s["noise"].gather(1, at).log()).masked_fill(~keep, -math.inf)
    won = race.argmax(-1, keepdim=True)
    won = torch.where(t > 0, won, 0)
    logp = d.gather(1, won) - w.sum(-1, keepdim=True).log()
    return dict(tok=at.gather(1, won)[:, 0].to(torch.int32), logp=torch.where(t > 0, logp, 0.0)[:, 0])


# ---- the work of a pass ----------------------------------------------------------


def work(case):
    if case["op"] == "sample":  # the logits, and the random numbers where no filter leaves most of them out
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (2 if case["bf16"] else 4) + (4 * n if case["kind"] == "none" else 0) + 24 * case["rows"], "flops": 4 * n}
    H, kv, hd = case["heads"], case["kv"], case["hd"]
    if case["op"] == "append":
        T = case["rows"]
        n = T * (H + 2 * kv) * hd * (4 if case["f32"] else 2) + T * H * hd * 2 + 2 * T * kv * _token_bytes(case) + 4 * T * case["rot"] + 8 * T
        if case["bits"] == 4:  # read back as values
            n += 2 * T * kv * (_token_bytes(case) + 2 * hd)
        return {"bytes": n, "flops": 8 * T * (H + kv) * hd}
    lens = _lengths(case)
    rows = sum(min(case["new"], n) for n in lens)
    pairs = sum(n * min(case["new"], n) for n in lens)
    return {"bytes": 2 * sum(lens) * kv * _token_bytes(case) + 4 * rows * H * hd, "flops": 4 * pairs * H * hd}


# ---- the same results in 64 bits -----------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    f = torch.float64
    if case["op"] == "sample":
        toks, logps = [], []
        for b in range(case["rows"]):
            row = s["logits"][b].to(f)
            order = torch.argsort(row, descending=True, stable=True)
            order = order[torch.isfinite(row[order])]
            T = float(s["temperature"][b])
            if T <= 0:
                toks.append(int(order[0]))
                logps.append(0.0)
                continue
            k = int(s["top_k"][b]) if s["top_k"] is not None else 0
            order = order[:k] if k > 0 else order
            z = (row[order] - row[order[0]]) / T
            mass = torch.exp(z)
            n = len(order)
            if s["top_p"] is not None and float(s["top_p"][b]) < 1:
                upto = torch.cumsum(mass, 0)
                n = 1 + int((upto[:-1] < s["top_p"][b].to(f) * upto[-1]).sum())
            if s["min_p"] is not None:
                n = min(n, max(1, int((mass >= s["min_p"][b].to(f)).sum())))
            score = z[:n] - torch.log(s["noise"][b][order[:n]].to(f))
            w = int(torch.argmax(score))
            toks.append(int(order[w]))
            logps.append(float(z[w] - torch.log(mass[:n].sum())))
        return dict(tok=torch.tensor(toks, dtype=torch.int32), logp=torch.tensor(logps, dtype=f))
    H, kv, hd, page = case["heads"], case["kv"], case["hd"], case["page"]
    if case["op"] == "append":
        x = s["qkv"].to(f).reshape(case["rows"], -1, hd)
        parts = [x[:, :H], x[:, H:H + kv]]
        if case["norm"]:
            parts = [t / torch.sqrt((t ** 2).sum(-1, keepdim=True) / hd + EPS) * w.to(f) for t, w in zip(parts, (s["g_q"], s["g_k"]))]
        if case["rot"]:
            j = torch.arange(case["rot"] // 2, device=x.device)
            i0, i1 = (2 * j, 2 * j + 1) if case["pairs"] else (j, j + case["rot"] // 2)
            turn = torch.complex(s["cos"].to(f), s["sin"].to(f))[s["pos"].long()][:, None]
            for t in range(2):
                y = parts[t].clone()
                z = torch.complex(y[..., i0], y[..., i1]) * turn
                y[..., i0], y[..., i1] = z.real, z.imag
                parts[t] = y
        k, v = parts[1], x[:, H + kv:]
        if case["bits"] == 16:
            pool = s["pool"].view(torch.bfloat16).to(f).reshape(-1, kv, 2, page, hd)
            slot = s["table"][s["seq"].long(), torch.div(s["pos"], page, rounding_mode="floor").long()].long()
            for part, t in enumerate((k, v)):
                pool[slot, :, part, s["pos"].long() % page] = t
            return dict(q=parts[0], pool=pool.reshape(s["pool"].shape[0], kv, -1))

        def held(t):  # a value in its group's sixteen steps; scale and minimum are kept in bf16
            y = t.reshape(*t.shape[:-1], hd // GROUP, GROUP)
            lo, hi = y.min(-1, keepdim=True).values, y.max(-1, keepdim=True).values
            step, base = ((hi - lo) / 15).to(torch.bfloat16).to(f), lo.to(torch.bfloat16).to(f)
            code = torch.where(step > 0, torch.clamp(torch.round((y - base) / step), 0, 15), 0.0)  # equal values: their minimum
            return (base + step * code).reshape(t.shape)

        return dict(q=parts[0], k=held(k), v=held(v))
    out, at, G = [], 0, H // kv
    for b, (n, rows) in enumerate(zip(_lengths(case), s["rows"])):
        blocks = s["pool"][s["table"][b, :-(-n // page)].long()].reshape(-1, kv, 2, page * _token_bytes(case))
        if case["bits"] == 16:
            x = blocks.view(torch.bfloat16).to(f).reshape(-1, kv, 2, page, hd)
        else:
            packed = blocks[..., :page * hd // 2].reshape(-1, kv, 2, page, hd // 2)
            mark = blocks[..., page * hd // 2:].contiguous().view(torch.bfloat16).to(f).reshape(-1, kv, 2, page, hd // GROUP, 2)
            x = torch.empty(*packed.shape[:-1], hd, dtype=f, device=packed.device)
            x[..., 0::2], x[..., 1::2] = (packed % 16).to(f), (packed // 16).to(f)
            x = x * mark[..., 0].repeat_interleave(GROUP, -1) + mark[..., 1].repeat_interleave(GROUP, -1)
        x = x.transpose(1, 3).reshape(-1, 2, kv, hd)[:n]  # tokens in order
        q = s["q"][at:at + rows].to(f).reshape(rows, kv, G, hd)
        z = torch.einsum("rkgd,nkd->rkgn", q, x[:, 0]) * s["scale"]
        seen = torch.arange(n, device=z.device)[None] <= torch.arange(n - rows, n, device=z.device)[:, None]
        z = torch.where(seen[:, None, None], z, -math.inf)
        out.append(torch.einsum("rkgn,nkd->rkgd", torch.softmax(z, -1), x[:, 1]).reshape(rows, H, hd))
        at += rows
    return torch.cat(out)
