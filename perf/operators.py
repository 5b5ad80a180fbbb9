"""The decoding operators as a user calls them, with a plain form of each for comparison.

Three operators of autoregressive decoding, measured over their real range:

* ``attend``  -- a chunk of new tokens (from one to thousands, another count per sequence) is written to a paged
  key / value cache and attends to everything the cache then holds (``paged_append`` + ``paged_attention``);
* ``select``  -- beam search's choice of the best continuations over beams and vocabulary (``beam_select``);
* ``reorder`` -- the page tables and half-filled pages of the beams that survive (``beam_reorder``).
"""
import math
import random

import torch

own = False

_DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


# ------------------------------------------------------------------------------------------------------ cases
def _attend(name, dtype, seqs, heads, kv_heads, dim, page, new, past, causal=True, append=True, mix=1):
    """`new` and `past` are (low, high): tokens per sequence in this call and in the cache before it; append: the new
    tokens' keys and values go into the cache first (not so where queries read another network's memory)"""
    return {"name": name, "op": "attend", "dtype": dtype, "seqs": seqs, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "page": page, "new_lo": new[0], "new_hi": new[1], "past_lo": past[0], "past_hi": past[1], "causal": causal,
            "append": append, "mix": mix}


def _select(name, dtype, batch, beams, vocab):
    return {"name": name, "op": "select", "dtype": dtype, "batch": batch, "beams": beams, "vocab": vocab}


def _reorder(name, dtype, batch, beams, layers, kv_heads, dim, page, past, mix=1):
    return {"name": name, "op": "reorder", "dtype": dtype, "batch": batch, "beams": beams, "layers": layers,
            "kv_heads": kv_heads, "dim": dim, "page": page, "past_lo": past[0], "past_hi": past[1], "mix": mix}


def listed():
    return [
        # one beam-search step of the stroke recognizer's masked self-attention: 32 images x 4 beams, 4 heads x 256, up to
        # 30 strokes so far -- a call whose latency counts
        _attend("strokes_step", "fp32", 128, 4, 4, 256, 16, (1, 1), (0, 29)),
        # its sibling's cross-attention: 4 beams of each of 128 images read that image's 256 positions, 16 heads x 64
        _attend("image_memory", "fp32", 128, 16, 16, 64, 16, (4, 4), (256, 256), causal=False, append=False),
        # one token each for 64 running sequences of very different lengths, grouped heads
        _attend("tokens_mixed", "bf16", 64, 32, 8, 128, 16, (1, 1), (100, 8190)),
        # one token each for two very long sequences: few rows, a long axis
        _attend("tokens_long", "bf16", 2, 32, 8, 128, 64, (1, 1), (131001, 131070)),
        # a scheduler's step: prompt chunks beside single tokens, odd lengths, some prompts at their start
        _attend("chunks_mixed", "bf16", 24, 32, 8, 128, 16, (1, 777), (0, 4000), mix=3),
        # short prompts of a small model: 16 heads x 64 without sharing
        _attend("prompts_small", "fp16", 37, 16, 16, 64, 32, (5, 300), (0, 0), mix=5),
        # the next 4096 tokens of one long document
        _attend("chunk_long", "bf16", 1, 32, 8, 128, 64, (4096, 4096), (12288, 12288)),
        # the stroke recognizer's alphabet: 32 images x 4 beams over 7 classes
        _select("select_strokes", "fp32", 32, 4, 7),
        # a character vocabulary of odd size
        _select("select_characters", "fp32", 64, 5, 6625),
        # a subword vocabulary in the logits' 16-bit type
        _select("select_subwords", "bf16", 64, 8, 50001),
        # the stroke recognizer's beams: little to move, latency counts
        _reorder("reorder_strokes", "fp32", 32, 4, 1, 4, 256, 16, (1, 30)),
        # 64 x 8 beams of a model with 4 layers and pages of 64 tokens
        _reorder("reorder_deep", "bf16", 64, 8, 4, 8, 128, 64, (20, 400)),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def _draw_once(rng):
    op = rng.choice(["attend", "attend", "attend", "attend", "select", "select", "reorder"])
    dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    dim = rng.choice([64, 128, 256])
    page = rng.choice([8, 16, 16, 32, 64, 128])
    mix = rng.randrange(1 << 30)
    if op == "attend":
        kv_heads, group = rng.choice([1, 2, 4, 8, 16]), rng.choice([1, 1, 2, 3, 4, 7, 8])
        kind = rng.choice(["token", "token", "chunk", "chunk", "memory"])
        seqs = _log_int(rng, 1, 256)
        if kind == "token":
            hi = _log_int(rng, 1, 131072)
            new, past, append = (1, 1), (rng.randrange(hi), hi), True
        elif kind == "memory":
            n = rng.choice([1, 2, 4, 5, 8])
            m = _log_int(rng, 16, 1024)
            new, past, append = (n, n), (m, m), False
        else:
            a, b = sorted((_log_int(rng, 1, 4096), _log_int(rng, 1, 4096)))
            p = rng.choice([0, _log_int(rng, 1, 16384)])
            new, past, append = (a, b), (rng.randrange(p + 1), p), True
        return _attend("", dtype, seqs, kv_heads * group, kv_heads, dim, page, new, past, append, append, mix)
    if op == "select":
        return _select("", dtype, _log_int(rng, 1, 128), rng.choice([1, 2, 3, 4, 5, 8, 10, 16]), _log_int(rng, 7, 200000))
    hi = _log_int(rng, 1, 4000)
    return _reorder("", dtype, _log_int(rng, 1, 128), rng.choice([2, 3, 4, 5, 8]), _log_int(rng, 1, 16),
                    rng.choice([1, 2, 4, 8]), dim, page, (rng.randrange(hi) + 1, hi), mix)


def draw(rng):
    """one more case of the listed ranges: no dearer than the dearest listed case of its operator"""
    top = {}
    for c in listed():
        w, t = work(c), top.setdefault(c["op"], {"bytes": 0, "flops": 0, "state": 0})
        # fp32 products run at a small part of the 16-bit rate, so they count for more
        t["flops"] = max(t["flops"], w["flops"] * (8 if c["dtype"] == "fp32" else 1))
        t["bytes"] = max(t["bytes"], w["bytes"])
    while True:
        c = _draw_once(rng)
        w, t = work(c), top[c["op"]]
        if c["op"] == "attend" and c["seqs"] * c["past_hi"] * c["kv_heads"] * c["dim"] > 1 << 29:
            continue                       # the padded plain form keeps keys and values in 32 bits
        if c["op"] == "reorder" and (c["batch"] * c["beams"] * c["layers"] * c["kv_heads"] * c["dim"]
                                     * (c["past_hi"] + 2 * c["page"])) * _SIZE[c["dtype"]] > 1 << 33:
            continue
        if w["bytes"] <= t["bytes"] and w["flops"] * (8 if c["dtype"] == "fp32" else 1) <= t["flops"]:
            del c["name"]
            return c


# --------------------------------------------------------------------------------------------------- lengths, work
def _lengths(case):
    """[(new, past)] of the sequences: a property of the case, spread over the given ranges"""
    rng = random.Random(case["mix"] * 1000003 + case["seqs"])
    out = []
    for _ in range(case["seqs"]):
        past = rng.randint(case["past_lo"], case["past_hi"])
        lo, hi = case["new_lo"], case["new_hi"]
        new = lo if lo == hi else (lo if rng.random() < 0.4 else _log_int(rng, max(1, lo), hi))
        out.append((new, past))
    return out


def _group_lengths(case):
    rng = random.Random(case["mix"] * 1000003 + case["batch"])
    return [rng.randint(case["past_lo"], case["past_hi"]) for _ in range(case["batch"])]


def work(case):
    es = _SIZE[case["dtype"]]
    if case["op"] == "attend":
        lens = _lengths(case)
        new, total = sum(n for n, _ in lens), sum(p for _, p in lens)
        if case["append"]:
            total, seen = total + new, sum(n * p + n * (n + 1) // 2 for n, p in lens)
        else:
            seen = sum(n * p for n, p in lens)
        kv = 2 * case["kv_heads"] * case["dim"] * es
        pages = sum(-(-(n + p) // case["page"]) for n, p in lens)
        written = new if case["append"] else 0
        # queries and outputs; the cache as it was is read, the new keys and values are read and written
        return {"bytes": 2 * new * case["heads"] * case["dim"] * es + (total + written) * kv + 4 * (pages + 2 * case["seqs"]),
                "flops": 4 * case["heads"] * case["dim"] * seen}
    if case["op"] == "select":
        rows = case["batch"] * case["beams"]
        # a subtraction, an exponential, an addition and a comparison per logit
        return {"bytes": rows * (case["vocab"] * es + 5 + 17), "flops": 4 * rows * case["vocab"]}
    lens, k = _group_lengths(case), case["beams"]
    row = 2 * case["layers"] * case["kv_heads"] * case["dim"] * es
    # parents are drawn evenly, the best beam stays where it is: k - 1 slots move with probability (k - 1) / k; a half-filled
    # page that several slots take over is read once
    rest = sum(n % case["page"] for n in lens)
    written = rest * (k - 1) * (k - 1) / k
    read = rest * ((1 - (1 - 1 / k) ** (k - 1)) + (k - 1) * (1 - (1 - 1 / k) ** (k - 2)))
    entries = sum(k * -(-(n + case["page"]) // case["page"]) for n in lens)
    return {"bytes": int((written + read) * row) + 8 * entries, "flops": 0}


# ----------------------------------------------------------------------------------------------------- prepare
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def prepare(case, seed):
    g, dt = _gen(seed), _DT[case["dtype"]]
    dev = torch.device("cuda")
    rnd = lambda *s: torch.randn(*s, generator=g, device=dev, dtype=torch.float32)             # noqa: E731
    if case["op"] == "attend":
        lens, page, dim = _lengths(case), case["page"], case["dim"]
        kvh, heads, seqs = case["kv_heads"], case["heads"], case["seqs"]
        kv = [n + p if case["append"] else p for n, p in lens]
        per_seq = -(-max(kv) // page)
        need = [-(-t // page) for t in kv]
        num_pages = sum(need) + 3
        # the pages of a sequence lie anywhere in the pool, as after some time of serving
        perm = torch.randperm(num_pages, generator=torch.Generator().manual_seed(seed)).tolist()
        table = torch.zeros(seqs, per_seq, dtype=torch.int32)
        at = 0
        for s, m in enumerate(need):
            table[s, :m] = torch.tensor(perm[at:at + m], dtype=torch.int32)
            at += m
        pool = lambda: torch.randn(num_pages, kvh, page, dim, generator=g, device=dev, dtype=torch.float32).to(dt)  # noqa: E731
        tokens = sum(n for n, _ in lens)
        st = {"case": case, "k_pages": pool(), "v_pages": pool(), "table": table.to(dev),
              "kv_lens": torch.tensor(kv, dtype=torch.int32, device=dev), "max_kv": max(kv),
              "max_q": max(n for n, _ in lens), "scale": 1.0 / math.sqrt(dim),
              "q": (1.5 * rnd(tokens, heads, dim)).to(dt), "k_new": rnd(tokens, kvh, dim).to(dt),
              "v_new": rnd(tokens, kvh, dim).to(dt), "q_start": None}
        # the first position of a prompt draws much of the attention
        first = st["table"][:, 0].long()
        st["k_pages"][first, :, 0] = (0.5 * st["k_pages"][first, :, 0].float() + 0.3).to(dt)
        if case["new_lo"] != case["new_hi"]:
            start = [0]
            for n, _ in lens:
                start.append(start[-1] + n)
            st["q_start"] = torch.tensor(start, dtype=torch.int32, device=dev)
        st["_lens"] = lens
        return st
    if case["op"] == "select":
        b, k, v = case["batch"], case["beams"], case["vocab"]
        x = 2.0 * rnd(b, k, v)
        # a trained model's distribution: a few likely continuations over a broad floor
        likely = torch.randint(0, v, (b, k, 6), generator=g, device=dev)
        x.scatter_add_(2, likely, 6.0 + 2.0 * rnd(b, k, 6).abs())
        scores = (-4.0 - 3.0 * rnd(b, k).abs()).sort(dim=1, descending=True).values.contiguous()
        finished = torch.rand(b, k, generator=g, device=dev) < 0.15
        if b > 2:
            scores[0, 1:] = float("-inf")            # a search at its first step: one beam holds all the weight
            finished[0] = False
        return {"case": case, "logits": x.to(dt), "scores": scores, "finished": finished, "eos": v - 1}
    b, k, page = case["batch"], case["beams"], case["page"]
    lens = _group_lengths(case)
    maxp = -(-max(lens) // page) + 1
    slots = b * k
    num_pages = slots * (maxp + 1)
    perm = torch.randperm(num_pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = perm[:slots * maxp].view(slots, maxp).contiguous().to(dev)
    spare = perm[slots * maxp:].contiguous().to(dev)
    parents = torch.randint(0, k, (b, k), generator=g, device=dev, dtype=torch.int32)
    parents[:, 0] = 0
    # beams share the full pages that they inherited from the best beam
    for i, n in enumerate(lens):
        table[i * k:(i + 1) * k, :n // page] = table[i * k, :n // page].clone()
    pool = torch.randint(-2 ** 15, 2 ** 15, (2 * case["layers"], num_pages, case["kv_heads"], page, case["dim"]),
                         generator=g, device=dev, dtype=torch.int16)
    pages = [(p.float() / 8192.0).to(dt) for p in pool]
    return {"case": case, "parents": parents, "table": table, "spare": spare, "pages": pages,
            "kv_lens": torch.tensor([n for n in lens for _ in range(k)], dtype=torch.int32, device=dev)}


# ------------------------------------------------------------------------------------------------------- own calls
def _run_own(st):
    from fudanocr_amd import decode as D
    case = st["case"]
    if case["op"] == "attend":
        cache = (st["k_pages"], st["v_pages"], st["table"], st["kv_lens"])
        if case["append"]:
            D.paged_append(st["k_new"], st["v_new"], *cache, q_start=st["q_start"])
        out = D.paged_attention(st["q"], *cache, q_start=st["q_start"], causal=case["causal"], scale=st["scale"],
                                max_q=st["max_q"], max_kv=st["max_kv"])
        return {"out": out, "k_pages": st["k_pages"], "v_pages": st["v_pages"]}
    if case["op"] == "select":
        scores, parents, tokens, finished = D.beam_select(st["logits"], st["scores"], st["finished"], eos=st["eos"])
        return {"scores": scores, "parents": parents, "tokens": tokens, "finished": finished}
    table, spare = D.beam_reorder(st["parents"], st["table"], st["kv_lens"], st["spare"], st["pages"])
    return {"table": table, "spare": spare, "pages": st["pages"]}


# ----------------------------------------------------------------------------------------------------- plain forms
def _append_plain(st):
    """positions of the new tokens -> (page, slot); the rows are written where a sequence's table says"""
    page, dev = st["case"]["page"], st["q"].device
    kv = st["kv_lens"].long()
    if st["q_start"] is None:
        n = st["q"].shape[0] // kv.numel()
        seq = torch.arange(kv.numel(), device=dev).repeat_interleave(n)
        first = torch.arange(kv.numel(), device=dev) * n
        count = torch.full_like(kv, n)
    else:
        start = st["q_start"].long()
        count = start[1:] - start[:-1]
        seq = torch.repeat_interleave(torch.arange(kv.numel(), device=dev), count, output_size=st["q"].shape[0])
        first = start[:-1]
    pos = kv[seq] - count[seq] + torch.arange(st["q"].shape[0], device=dev) - first[seq]
    pg = st["table"][seq, pos // page].long()
    st["k_pages"][pg, :, pos % page] = st["k_new"]
    st["v_pages"][pg, :, pos % page] = st["v_new"]


def _gather(pages, table, length):
    """[S, Hkv, length, D] in 32 bits: the cache of every sequence in order (past a sequence's end: whatever is there)"""
    page = pages.shape[2]
    m = -(-length // page)
    x = pages[table[:, :m].long()].float()                                # [S, m, Hkv, page, D]
    return x.permute(0, 2, 1, 3, 4).reshape(x.shape[0], x.shape[2], m * page, x.shape[4])[:, :, :length]


def _softmax_product(q, k, v, visible, scale):
    """q [.., R, D], k / v [.., L, D], visible [.., R, L] -> [.., R, D]; rows that see nothing are zero"""
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) * scale
    s = s.masked_fill(~visible, float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isfinite(m), m, torch.zeros_like(m)))
    return torch.matmul(p, v) / p.sum(-1, keepdim=True).clamp_min(1e-37)


def _attend_plain(st):
    case, lens = st["case"], st["_lens"]
    if case["append"]:
        _append_plain(st)
    heads, kvh, dim = case["heads"], case["kv_heads"], case["dim"]
    grp, dev = heads // kvh, st["q"].device
    q, out = st["q"].float(), torch.empty_like(st["q"])
    if st["q_start"] is None and st["max_q"] <= 16:
        n, seqs, length = st["max_q"], case["seqs"], st["max_kv"]
        k, v = _gather(st["k_pages"], st["table"], length), _gather(st["v_pages"], st["table"], length)
        pos = torch.arange(length, device=dev)
        kv = st["kv_lens"].long()
        last = kv[:, None] - n + torch.arange(n, device=dev) if case["causal"] else (kv[:, None] - 1).expand(seqs, n)
        vis = pos <= last[..., None]                                      # [S, n, L]
        vis = vis[:, None, None].expand(seqs, 1, grp, n, length).reshape(seqs, 1, grp * n, length)
        v = v.masked_fill((pos >= kv[:, None])[:, None, :, None], 0.0)
        qs = q.view(seqs, n, kvh, grp, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kvh, grp * n, dim)
        o = _softmax_product(qs, k, v, vis, st["scale"])
        o = o.view(seqs, kvh, grp, n, dim).permute(0, 3, 1, 2, 4).reshape(seqs * n, heads, dim)
        return {"out": o.to(st["q"].dtype), "k_pages": st["k_pages"], "v_pages": st["v_pages"]}
    at = 0
    for s, (n, past) in enumerate(lens):
        length = n + past if case["append"] else past
        k, v = (_gather(st[x], st["table"][s:s + 1], length)[0] for x in ("k_pages", "v_pages"))
        vis = torch.arange(length, device=dev) <= (past + torch.arange(n, device=dev))[:, None] if case["causal"] \
            else torch.ones(n, length, dtype=torch.bool, device=dev)
        qs = q[at:at + n].view(n, kvh, grp, dim).permute(1, 2, 0, 3).reshape(kvh, grp * n, dim)
        o = _softmax_product(qs, k, v.contiguous(), vis.repeat(grp, 1), st["scale"])
        out[at:at + n] = o.view(kvh, grp, n, dim).permute(2, 0, 1, 3).reshape(n, heads, dim).to(out.dtype)
        at += n
    return {"out": out, "k_pages": st["k_pages"], "v_pages": st["v_pages"]}


def _candidates(logits, scores, finished, eos):
    """[B, K, V] candidate scores in 64 bits (two beams' continuations may differ by less than 32 bits hold)"""
    x = logits.double()
    norm = torch.logsumexp(x, dim=2, keepdim=True)
    live = torch.isfinite(norm) & torch.isfinite(scores)[..., None]
    ended = torch.full_like(x, float("-inf"))
    ended[..., eos] = scores.double()
    cand = torch.where(finished[..., None], ended, scores.double()[..., None] + (x - norm))
    dead = torch.where(finished, ~torch.isfinite(scores), ~live[..., 0])[..., None]
    return torch.where(dead | torch.isnan(cand), torch.full_like(cand, float("-inf")), cand)


def _best(cand, finished, eos):
    b, k, v = cand.shape
    val, idx = torch.sort(cand.view(b, k * v), dim=1, descending=True, stable=True)
    val, idx = val[:, :k], idx[:, :k]
    parents, tokens = idx // v, idx % v
    return val, parents.int(), tokens, torch.gather(finished, 1, parents) | (tokens == eos)


def _select_plain(st):
    cand = _candidates(st["logits"], st["scores"], st["finished"], st["eos"])
    val, parents, tokens, finished = _best(cand, st["finished"], st["eos"])
    return {"scores": val.float(), "parents": parents, "tokens": tokens, "finished": finished}


def _reorder_plain(st):
    case = st["case"]
    k, page, dev = case["beams"], case["page"], st["table"].device
    b, maxp = case["batch"], st["table"].shape[1]
    slots = torch.arange(b * k, device=dev)
    src = (slots // k) * k + st["parents"].long().view(-1)
    n = st["kv_lens"].long()
    full, rest = n // page, n % page
    col = torch.arange(maxp, device=dev)
    table = torch.where(col < full[:, None], st["table"][src], st["table"])
    move = (src != slots) & (rest > 0)
    at = full.clamp_max(maxp - 1)
    old = st["table"][slots, at]
    table[slots, at] = torch.where(move, st["spare"], table[slots, at])
    spare = torch.where(move, old, st["spare"])
    from_page, to_page = st["table"][src, at].long(), st["spare"].long()
    slot = torch.arange(page, device=dev)
    who, row = torch.nonzero(move[:, None] & (slot < rest[:, None]), as_tuple=True)
    for p in st["pages"]:
        p[to_page[who], :, row] = p[from_page[who], :, row]
    return {"table": table, "spare": spare, "pages": st["pages"]}


def run(state):
    if own:
        return _run_own(state)
    return {"attend": _attend_plain, "select": _select_plain, "reorder": _reorder_plain}[state["case"]["op"]](state)


# ----------------------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    """the operators' definitions in 64 bits, one sequence and head (one batch entry) at a time"""
    st = prepare(case, seed)
    dev = torch.device("cuda")
    if case["op"] == "reorder":                       # nothing is computed: rows and whole numbers move
        table, spare, lens = st["table"].tolist(), st["spare"].tolist(), st["kv_lens"].tolist()
        parents, k, page = st["parents"].flatten().tolist(), case["beams"], case["page"]
        new_table, new_spare = [list(r) for r in table], list(spare)
        for j, n in enumerate(lens):
            p = j // k * k + parents[j]
            new_table[j][:n // page] = table[p][:n // page]
            if n % page and p != j:
                new_table[j][n // page], new_spare[j] = spare[j], table[j][n // page]
                for x in st["pages"]:
                    x[spare[j], :, :n % page] = x[table[p][n // page], :, :n % page]
        return {"table": torch.tensor(new_table, dtype=torch.int32, device=dev),
                "spare": torch.tensor(new_spare, dtype=torch.int32, device=dev), "pages": st["pages"]}
    if case["op"] == "select":
        b, k, v = case["batch"], case["beams"], case["vocab"]
        val = torch.empty(b, k, dtype=torch.float64, device=dev)
        parents, tokens = (torch.empty(b, k, dtype=torch.int64, device=dev) for _ in range(2))
        for i in range(b):
            x = st["logits"][i].double()
            top = x.amax(1, keepdim=True)
            logp = x - top - torch.exp(x - top).sum(1, keepdim=True).log()
            cand = st["scores"][i].double()[:, None] + logp
            for j in torch.nonzero(st["finished"][i]).flatten().tolist():
                cand[j] = float("-inf")
                cand[j, st["eos"]] = st["scores"][i, j].double()
            flat = torch.nan_to_num(cand, nan=float("-inf"), neginf=float("-inf")).flatten()
            for r in range(k):                        # the largest that is left; among equals the first
                best = flat.amax()
                at = torch.nonzero(flat == best)[0, 0] if torch.isfinite(best) else None
                if at is None:
                    break
                val[i, r], parents[i, r], tokens[i, r] = best, at // v, at % v
                flat[at] = float("nan")
                flat = torch.nan_to_num(flat, nan=float("-inf"), neginf=float("-inf"))
            else:
                continue
            return None                               # fewer live continuations than beams: no 64-bit value for the rest
        fin = torch.gather(st["finished"], 1, parents) | (tokens == st["eos"])
        return {"scores": val, "parents": parents, "tokens": tokens, "finished": fin}
    if work(case)["flops"] > 4e12:
        return None
    heads, kvh, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    grp = heads // kvh
    out = torch.empty(st["q"].shape, dtype=torch.float64, device=dev)
    table, at = st["table"].cpu(), 0
    for s, (n, past) in enumerate(st["_lens"]):
        length = n + past if case["append"] else past
        ids = table[s, :-(-length // page)].long().to(dev)
        for h in range(kvh):
            k, v = (torch.cat([st[c][ids, h].reshape(-1, dim)[:past], st[w][at:at + length - past, h]]).double()
                    for c, w in (("k_pages", "k_new"), ("v_pages", "v_new")))
            for i in range(0, n, 1024):
                m = min(1024, n - i)
                q = st["q"][at + i:at + i + m, h * grp:(h + 1) * grp].double()                 # [m, G, D]
                w = (q.reshape(m * grp, dim) @ k.t()).view(m, grp, -1) * st["scale"]
                if case["causal"]:
                    late = torch.arange(length, device=dev) > (past + i + torch.arange(m, device=dev))[:, None]
                    w.masked_fill_(late[:, None], float("-inf"))
                w = torch.exp(w - w.amax(-1, keepdim=True))
                o = (w / w.sum(-1, keepdim=True)).view(m * grp, -1) @ v
                out[at + i:at + i + m, h * grp:(h + 1) * grp] = o.view(m, grp, dim)
        at += n
    return {"out": out, "k_pages": None, "v_pages": None}
