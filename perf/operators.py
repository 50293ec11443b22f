"""Cases for measuring the serving operators of streams that share a prompt:

  plan    block tables, slot map, positions and row map of a step from the streams' lengths
  write   new K and V rows into cache pages by the slot map
  attend  one query token per stream over a shared prefix and the stream's own pages
  sample  one token per row from logits: temperature, min-p, top-k, top-p, given random numbers

``run`` computes an operator in its plain form (``own`` false) or calls the framework's.
"""
import math

import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
ONE = 2.0 ** 44  # fixed-point weight of a row's largest logit


def listed():
    return [
        # one decode step of 64 streams: a token each, a new page now and then
        dict(name="plan_decode_64", op="plan", streams=64, new_lo=1, new_hi=1, own_lo=0, own_hi=4095, page=16, prefix=2048),
        # admission of 64 prompts of very different lengths in one packed batch
        dict(name="plan_prompts_64", op="plan", streams=64, new_lo=16, new_hi=16384, own_lo=0, own_hi=0, page=64, prefix=0),
        # the step's new K/V rows of 64 streams, from the f32 activations of the projections
        dict(name="write_step_64", op="write", tokens=64, nkv=8, dim=256, src="f32", dst="f16", page=16, pages=2048),
        # a packed prompt chunk, K and V as slices of the fused q|k|v projection
        dict(name="write_prompt_8k", op="write", tokens=8191, nkv=8, dim=256, src="bf16", dst="bf16", page=32, pages=512),
        # a few streams right after a short system prompt: latency
        dict(name="attend_small_4", op="attend", streams=4, prefix=192, own_lo=1, own_hi=32, nq=4, nkv=2, dim=256, page=16, window=0, type="f16"),
        # full-attention layer of a 64-stream step behind a 4K-token shared prompt
        dict(name="attend_4k_64", op="attend", streams=64, prefix=4096, own_lo=1, own_hi=1023, nq=16, nkv=8, dim=256, page=16, window=0, type="f16"),
        # the same with a very long shared document
        dict(name="attend_32k_64", op="attend", streams=64, prefix=32768, own_lo=1, own_hi=2047, nq=16, nkv=8, dim=256, page=64, window=0, type="bf16"),
        # sliding-window layer: long streams no longer see the prompt, fresh ones see part of it
        dict(name="attend_window_64", op="attend", streams=64, prefix=2000, own_lo=0, own_hi=1500, nq=16, nkv=8, dim=256, page=16, window=1024, type="bf16"),
        # odd batch, ragged prefix, smaller heads with four queries per kv head
        dict(name="attend_gqa4_37", op="attend", streams=37, prefix=1001, own_lo=0, own_hi=777, nq=32, nkv=8, dim=128, page=32, window=0, type="f16"),
        # one stream's token from the full 262,144-entry head
        dict(name="sample_1", op="sample", rows=1, vocab=262144, pad=0, type="f32", softcap=30.0, mix="all"),
        # a 64-stream step, every stream with its own settings, greedy ones among them
        dict(name="sample_64", op="sample", rows=64, vocab=262144, pad=0, type="f32", softcap=30.0, mix="mixed"),
        # rows of a padded 16-bit logits buffer, an odd vocabulary, top-p and min-p only
        dict(name="sample_bf16_48", op="sample", rows=48, vocab=100003, pad=61, type="bf16", softcap=0.0, mix="mass"),
    ]


def log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "write", "attend", "attend", "attend", "sample", "sample"])
    if op == "plan":
        streams = log_int(rng, 1, 512)
        if rng.random() < 0.5:
            lo, hi, own_hi = 1, 1, log_int(rng, 1, 8000)
        else:
            lo, hi, own_hi = 1, log_int(rng, 2, 16384 if streams <= 64 else (1 << 20) // streams), rng.choice([0, 777])
        return dict(op=op, streams=streams, new_lo=lo, new_hi=hi, own_lo=0, own_hi=own_hi, page=rng.choice([16, 32, 64, 128]), prefix=rng.choice([0, 100, 2048]))
    if op == "write":
        nkv, dim = rng.choice([(8, 256), (2, 256), (1, 256), (8, 128), (4, 64)])
        src, dst = rng.choice([("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
        tokens, page = log_int(rng, 1, 8191), rng.choice([16, 32, 64])
        return dict(op=op, tokens=tokens, nkv=nkv, dim=dim, src=src, dst=dst, page=page, pages=max(64, 2 * tokens // page))
    if op == "attend":
        nq, nkv, dim = rng.choice([(16, 8, 256), (8, 1, 256), (4, 2, 256), (32, 8, 128), (8, 8, 128), (16, 4, 64)])
        return dict(op=op, streams=log_int(rng, 1, 64), prefix=rng.choice([0, 1, 1, 1]) * log_int(rng, 1, 32768), own_lo=rng.choice([0, 1]),
                    own_hi=log_int(rng, 1, 2047), nq=nq, nkv=nkv, dim=dim, page=rng.choice([16, 32, 64]),
                    window=rng.choice([0, 0, 0, 1]) * log_int(rng, 1, 2048), type=rng.choice(["f16", "bf16"]))
    return dict(op=op, rows=log_int(rng, 1, 64), vocab=log_int(rng, 500, 262144), pad=rng.choice([0, 0, 1, 61]), type=rng.choice(["f32", "f32", "bf16", "f16"]),
                softcap=rng.choice([0.0, 30.0]), mix=rng.choice(["all", "mixed", "mass", "plain"]))


def ragged(lo, hi, n):
    """n lengths spread evenly over [lo, hi]; a case has the same ones for every seed."""
    return [lo + int((hi - lo) * (i + 0.5) / n + 0.5) for i in range(n)]


def shuffled(values, g):
    order = torch.randperm(len(values), generator=g, device=DEV)
    return torch.tensor(values, dtype=torch.int32, device=DEV)[order]


def pages_of(lens, page):
    return [(n + page - 1) // page for n in lens]


def new_tables(lens, page, blocks, pages, g, first=0):
    """Block tables of streams whose pages lie anywhere in the pool (the pages past the first `first`)."""
    free = torch.randperm(pages - first, generator=g, device=DEV).int() + first
    need = (lens + page - 1) // page
    end = torch.cumsum(need, 0)
    at = (end - need)[:, None] + torch.arange(blocks, device=DEV)
    table = free[at.clamp(max=len(free) - 1)]
    table[torch.arange(blocks, device=DEV) >= need[:, None]] = -1
    return table.int(), free[int(end[-1]):]


def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(int(seed))
    s = dict(case)
    if case["op"] == "plan":
        n, page = case["streams"], case["page"]
        old = ragged(case["own_lo"], case["own_hi"], n)
        new = ragged(case["new_lo"], case["new_hi"], n)
        blocks = (max(old) + max(new) + page - 1) // page + 1
        s["max_tokens"] = sum(new)
        s["lens"], s["new"] = shuffled(old, g), shuffled(new, g)
        spare = sum(pages_of(new, page)) + n
        s["table"], free = new_tables(s["lens"], page, blocks, sum(pages_of(old, page)) + spare, g)
        s["free"] = free.contiguous()
    elif case["op"] == "write":
        n, nkv, dim = case["tokens"], case["nkv"], case["dim"]
        # k and v as a program has them: slices of the fused q|k|v projection
        qkv = torch.randn(n, 4 * nkv * dim, generator=g, device=DEV, dtype=TYPES[case["src"]])
        s["k"] = qkv[:, 2 * nkv * dim:3 * nkv * dim].view(n, nkv, dim)
        s["v"] = qkv[:, 3 * nkv * dim:].view(n, nkv, dim)
        shape = (case["pages"], case["page"], nkv, dim)
        s["k_pool"] = torch.randn(shape, generator=g, device=DEV, dtype=TYPES[case["dst"]])
        s["v_pool"] = torch.randn(shape, generator=g, device=DEV, dtype=TYPES[case["dst"]])
        s["slots"] = torch.randperm(case["pages"] * case["page"], generator=g, device=DEV)[:n].int()
        if n > 4:  # padding at the end of a packed batch
            s["slots"][-2:] = -1
    elif case["op"] == "attend":
        n, page, t = case["streams"], case["page"], TYPES[case["type"]]
        lens = ragged(case["own_lo"], case["own_hi"], n)
        shared = (case["prefix"] + page - 1) // page
        pages = shared + sum(pages_of(lens, page)) + 8
        shape = (pages, page, case["nkv"], case["dim"])
        s["k_pool"] = torch.randn(shape, generator=g, device=DEV, dtype=t)
        s["v_pool"] = torch.randn(shape, generator=g, device=DEV, dtype=t)
        # scores with a spread of about 2.5, as normalised heads have
        s["q"] = (2.5 * torch.randn(n, case["nq"], case["dim"], generator=g, device=DEV)).to(t)
        s["lens"] = shuffled(lens, g)
        s["prefix_table"] = torch.randperm(max(shared, 1), generator=g, device=DEV).int()[:shared]
        blocks = max(1, (max(lens) + page - 1) // page)
        s["table"], _ = new_tables(s["lens"], page, blocks, pages, g, shared)
        s["scale"] = case["dim"] ** -0.5
    else:
        n, vocab = case["rows"], case["vocab"]
        # a broad body and a few dozen likely tokens per row
        x = 2.0 * torch.randn(n, vocab + case["pad"], generator=g, device=DEV)
        top = torch.randint(0, vocab, (n, 48), generator=g, device=DEV)
        x.scatter_add_(1, top, 12.0 * torch.rand(n, 48, generator=g, device=DEV).sqrt() + 2.0)
        s["logits"] = x.to(TYPES[case["type"]])[:, :vocab]
        s["uniform"] = torch.rand(n, generator=g, device=DEV)

        def pick(values, kind):
            at = torch.randint(0, len(values), (n,), generator=g, device=DEV)
            return torch.tensor(values, dtype=kind, device=DEV)[at]

        mix = case["mix"]
        s["temperature"] = pick([0.0, 0.6, 0.8, 1.0, 1.3] if mix == "mixed" else [0.7, 1.0, 1.2], torch.float32)
        s["top_k"] = pick([64], torch.int32) if mix == "all" else pick([0, 20, 64, 1000], torch.int32) if mix == "mixed" else None
        s["top_p"] = None if mix == "plain" else pick([0.95], torch.float32) if mix == "all" else pick([0.8, 0.9, 0.95, 1.0], torch.float32)
        s["min_p"] = None if mix == "plain" else pick([0.0, 0.02, 0.05] if mix != "all" else [0.05], torch.float32)
    return s


# ---- plain forms ---------------------------------------------------------------


def plain_plan(s):
    lens, new, page, table, free = s["lens"].long(), s["new"].long(), s["page"], s["table"].long(), s["free"].long()
    blocks = table.shape[1]
    have = (lens + page - 1) // page
    after = ((lens + new + page - 1) // page).clamp(max=blocks)
    fresh = (after - have).clamp(min=0)
    starts = torch.cat([new.new_zeros(1), torch.cumsum(new, 0)])
    first = torch.cumsum(fresh, 0) - fresh
    column = torch.arange(blocks, device=DEV)[None]
    rank = first[:, None] + column - have[:, None]
    padded = torch.cat([free, free.new_full((1,), -1)])
    page_of = padded[rank.clamp(min=0, max=len(free))]
    table = torch.where((column >= have[:, None]) & (column < after[:, None]), page_of, table)
    t = torch.arange(s["max_tokens"], device=DEV)
    there = t < starts[-1]
    row = torch.searchsorted(starts[1:].contiguous(), t, right=True).clamp(max=len(lens) - 1)
    i = lens[row] + t - starts[row]
    block = i // page
    at = table[row, block.clamp(max=blocks - 1)]
    slot = torch.where(there & (block < blocks) & (at >= 0), at * page + i % page, -1)
    out = dict(table=table, lens=lens + new, starts=starts, slots=slot, positions=torch.where(there, s["prefix"] + i, -1),
               rows=torch.where(there, row, -1), counts=torch.stack([starts[-1], fresh.sum()]))
    return {k: v.int() for k, v in out.items()}


def plain_write(s):
    keep = s["slots"] >= 0
    at = s["slots"][keep].long()
    for pool, x in ((s["k_pool"], s["k"]), (s["v_pool"], s["v"])):
        pool.view(-1, *pool.shape[2:])[at] = x[keep].float().to(pool.dtype)
    return dict(k_pool=s["k_pool"], v_pool=s["v_pool"])


def plain_attend(s):
    n, nq, dim = s["q"].shape
    page, nkv, prefix = s["page"], s["nkv"], s["prefix"]
    group = nq // nkv
    k_rows, v_rows = (s[p].view(-1, nkv, dim) for p in ("k_pool", "v_pool"))
    q = s["q"].float().view(n, nkv, group, dim) * s["scale"]
    lens = s["lens"].long()
    low = (prefix + lens - s["window"]).clamp(min=0) if s["window"] else torch.zeros_like(lens)

    def rows_of(table, count):
        i = torch.arange(count, device=DEV)
        return table[..., i // page].clamp(min=0).long() * page + i % page

    # scores over the shared prefix (a product over all streams) and over each stream's own tokens
    shared = rows_of(s["prefix_table"], prefix)
    a = torch.einsum("nhgd,phd->nhgp", q, k_rows[shared].float())
    a = a.masked_fill((torch.arange(prefix, device=DEV) < low[:, None])[:, None, None], -math.inf)
    width = s["table"].shape[1] * page
    mine = rows_of(s["table"], width)
    b = torch.einsum("nhgd,nihd->nhgi", q, k_rows[mine].float())
    i = torch.arange(width, device=DEV)
    b = b.masked_fill(((i >= lens[:, None]) | (i + prefix < low[:, None]))[:, None, None], -math.inf)
    scores = torch.cat([a, b], -1)
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    o = torch.einsum("nhgp,phd->nhgd", p[..., :prefix], v_rows[shared].float())
    o = o + torch.einsum("nhgi,nihd->nhgd", p[..., prefix:], v_rows[mine].float())
    o = torch.where(total > 0, o / total, 0.0)
    return o.reshape(n, nq, dim).to(s["q"].dtype)


def plain_sample(s):
    x = s["logits"].float()
    n, vocab = x.shape
    if s["softcap"]:
        x = torch.tanh(x / torch.full_like(x[:, :1], s["softcap"])) * s["softcap"]
    top, best = x.max(1, keepdim=True)
    best = (x == top).long().argmax(1)
    cold = s["temperature"] <= 0
    t = torch.where(cold, 1.0, s["temperature"])[:, None]
    e = torch.exp(torch.where(x == top, 0.0, (x - top) / t))
    w = (e * ONE).to(torch.int64)
    # by weight, equal ones by index; every filter keeps a first part of this order
    e, order = torch.sort(e, dim=1, descending=True, stable=True)
    w_sorted = w.gather(1, order)
    keep = w_sorted > 0
    if s["min_p"] is not None:
        keep &= (e >= s["min_p"][:, None]) | (e == 1)
    if s["top_k"] is not None:
        k = torch.where(s["top_k"] > 0, s["top_k"], vocab)[:, None]
        keep &= torch.arange(vocab, device=DEV) < k
    if s["top_p"] is not None:
        w_kept = torch.where(keep, w_sorted, 0)
        mass = torch.cumsum(w_kept, 1)
        p = s["top_p"].double()[:, None]
        need = torch.ceil(p * mass[:, -1:].double()).to(torch.int64).clamp(min=1)
        keep &= (mass - w_kept < need) | (p >= 1)
    kept = keep.sum(1)
    mask = torch.zeros_like(keep).scatter(1, order, keep)
    run_mass = torch.cumsum(torch.where(mask, w, 0), 1)
    total = run_mass[:, -1]
    goal = torch.minimum((s["uniform"].double() * total.double()).to(torch.int64), total - 1)
    token = (run_mass <= goal[:, None]).sum(1)
    token = torch.where(cold, best, token.clamp(max=vocab - 1))
    share = torch.log(w.gather(1, token[:, None])[:, 0].double() / total.double())
    return dict(tokens=token.int(), logprobs=torch.where(cold, 0.0, share).float(), kept=torch.where(cold, 1, kept).int())


def run(state):
    s = state
    if not own:
        return {"plan": plain_plan, "write": plain_write, "attend": plain_attend, "sample": plain_sample}[s["op"]](s)
    if s["op"] == "sample":
        from channel_b200 import sampling
        tokens, logprobs, kept = sampling.sample_rows(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                                                      min_p=s["min_p"], softcap=s["softcap"])
        return dict(tokens=tokens, logprobs=logprobs, kept=kept)
    from channel_b200 import paged
    if s["op"] == "plan":
        p = paged.plan_pages(s["lens"], s["new"], s["table"], s["free"], s["page"], s["max_tokens"], prefix_len=s["prefix"])
        return dict(table=p.table, lens=p.lens, starts=p.starts, slots=p.slots, positions=p.positions, rows=p.rows, counts=p.counts)
    if s["op"] == "write":
        paged.kv_write(s["k"], s["v"], s["slots"], s["k_pool"], s["v_pool"])
        return dict(k_pool=s["k_pool"], v_pool=s["v_pool"])
    return paged.prefix_attention(s["q"], s["k_pool"], s["v_pool"], s["table"], s["lens"], prefix_table=s["prefix_table"], prefix_len=s["prefix"],
                                  window=s["window"], scale=s["scale"])


# ---- what a pass cannot do without ------------------------------------------------


def work(case):
    if case["op"] == "plan":
        n, page = case["streams"], case["page"]
        old, new = ragged(case["own_lo"], case["own_hi"], n), ragged(case["new_lo"], case["new_hi"], n)
        tokens, pages = sum(new), sum(new) // page + n // 2
        return dict(bytes=4 * (3 * tokens + 2 * pages + 5 * n) + 12, flops=0)
    if case["op"] == "write":
        return dict(bytes=2 * case["tokens"] * case["nkv"] * case["dim"] * (SIZE[case["src"]] + SIZE[case["dst"]]) + 4 * case["tokens"], flops=0)
    if case["op"] == "attend":
        lens, prefix, window = ragged(case["own_lo"], case["own_hi"], case["streams"]), case["prefix"], case["window"] or 1 << 40
        seen_prefix = [max(0, prefix - max(0, prefix + n - window)) for n in lens]
        seen_own = [min(n, window) for n in lens]
        rows = max(seen_prefix) + sum(seen_own)
        row = case["dim"] * SIZE[case["type"]]
        return dict(bytes=2 * rows * case["nkv"] * row + 2 * case["streams"] * case["nq"] * row + 4 * (rows // case["page"] + case["streams"]),
                    flops=4 * case["nq"] * case["dim"] * (sum(seen_prefix) + sum(seen_own)))
    return dict(bytes=case["rows"] * (case["vocab"] * SIZE[case["type"]] + 32), flops=0)


# ---- the definitions in 64 bits ------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "plan":
        return None  # whole numbers only
    if case["op"] == "write":
        out = {}
        for name, src in (("k_pool", "k"), ("v_pool", "v")):
            pool = s[name].double().flatten(0, 1)
            for t, slot in enumerate(s["slots"].tolist()):
                if slot >= 0:
                    pool[slot] = s[src][t].double()
            out[name] = pool.view(s[name].shape)
        return out
    if case["op"] == "attend":
        n, nq, dim = s["q"].shape
        page, group = s["page"], nq // s["nkv"]
        out = torch.zeros(n, nq, dim, dtype=torch.float64, device=DEV)
        for b, length in enumerate(s["lens"].tolist()):
            k = [p[s["prefix_table"].long()].flatten(0, 1)[:s["prefix"]] for p in (s["k_pool"], s["v_pool"])]
            used = s["table"][b, :(length + page - 1) // page].long()
            mine = [p[used].flatten(0, 1)[:length] for p in (s["k_pool"], s["v_pool"])]
            keys, values = (torch.cat(x)[-s["window"] if s["window"] else 0:].double() for x in zip(k, mine))
            if not len(keys):
                continue
            for h in range(s["nkv"]):
                z = s["q"][b, h * group:(h + 1) * group].double() @ keys[:, h].T * s["scale"]
                out[b, h * group:(h + 1) * group] = torch.softmax(z, 1) @ values[:, h]
        return out
    logprobs = []
    for r in range(case["rows"]):
        x = s["logits"][r].double()
        if s["softcap"]:
            x = s["softcap"] * torch.tanh(x / s["softcap"])
        t = float(s["temperature"][r])
        if t <= 0:
            logprobs.append(0.0)
            continue
        p = torch.exp((x - x.max()) / t)
        down, order = torch.sort(p, descending=True, stable=True)
        count = len(p)
        if s["min_p"] is not None:
            count = max(1, int((down >= float(s["min_p"][r])).sum()))
        if s["top_k"] is not None and int(s["top_k"][r]) > 0:
            count = min(count, int(s["top_k"][r]))
        if s["top_p"] is not None and float(s["top_p"][r]) < 1:
            mass = torch.cumsum(down[:count], 0)
            count = int((mass - down[:count] < float(s["top_p"][r]) * mass[-1]).sum())
        stay = torch.zeros_like(p)
        stay[order[:count]] = down[:count]
        mass = torch.cumsum(stay, 0)
        token = int(torch.searchsorted(mass, float(s["uniform"][r]) * mass[-1], right=True))
        logprobs.append(math.log(float(stay[token] / mass[-1])))
    return dict(tokens=None, logprobs=torch.tensor(logprobs, dtype=torch.float64), kept=None)
