"""Cases for measuring the operators of steps with several tokens per stream:

  prompt  causal attention of packed prompts (or prompt chunks), each over its cached tokens and itself
  tree    attention of trees of drafted tokens over their streams' caches
  score   log-probability, entropy, rank and top alternatives of given tokens, from logits rows
  accept  which drafted tokens of each stream's tree the sampled ones confirm

``run`` computes an operator in its plain form (``own`` false) or calls the framework's.
"""
import math

import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # a short question to a small model: latency
        dict(name="prompt_9", op="prompt", streams=1, new_lo=9, new_hi=9, prefix=0, old_lo=0, old_hi=0, nq=4, nkv=2, dim=256, page=16, window=0, type="f16", pad=0),
        # admission of 64 prompts of very different lengths in one packed batch, a sliding-window layer
        dict(name="prompts_64", op="prompt", streams=64, new_lo=16, new_hi=2048, prefix=0, old_lo=0, old_hi=0, nq=16, nkv=8, dim=256, page=16, window=1024, type="bf16", pad=0),
        # one long document, a full-attention layer
        dict(name="prompt_16k", op="prompt", streams=1, new_lo=16384, new_hi=16384, prefix=0, old_lo=0, old_hi=0, nq=16, nkv=8, dim=256, page=16, window=0, type="f16", pad=0),
        # chunks of ragged prompts behind their cached part and a shared system prompt, smaller heads, a padded batch
        dict(name="chunks_21", op="prompt", streams=21, new_lo=1, new_hi=999, prefix=1001, old_lo=0, old_hi=4095, nq=32, nkv=8, dim=128, page=32, window=0, type="bf16", pad=61),
        # one stream's few drafted tokens: latency
        dict(name="tree_1", op="tree", streams=1, new_lo=8, new_hi=8, prefix=0, old_lo=300, old_hi=300, nq=16, nkv=8, dim=256, page=16, window=0, type="f16", pad=0),
        # a 64-stream step with 16 drafted tokens each
        dict(name="tree_64", op="tree", streams=64, new_lo=16, new_hi=16, prefix=0, old_lo=1, old_hi=4095, nq=16, nkv=8, dim=256, page=16, window=0, type="f16", pad=0),
        # trees of very different sizes on one kv head, behind a shared prompt, a window across both
        dict(name="tree_mqa_37", op="tree", streams=37, new_lo=1, new_hi=61, prefix=1001, old_lo=0, old_hi=2047, nq=8, nkv=1, dim=256, page=64, window=1024, type="bf16", pad=0),
        # one row: latency of reading 1 MB
        dict(name="score_1", op="score", rows=1, vocab=262144, pad=0, type="f32", softcap=30.0, top=20),
        # the tokens of a 512-token prompt
        dict(name="score_512", op="score", rows=512, vocab=262144, pad=0, type="f32", softcap=30.0, top=5),
        # rows of a padded 16-bit logits buffer, an odd vocabulary
        dict(name="score_bf16_777", op="score", rows=777, vocab=100003, pad=61, type="bf16", softcap=0.0, top=20),
        # the step of tree_64
        dict(name="accept_64", op="accept", streams=64, new_lo=16, new_hi=16),
        # a large batch of small and large trees
        dict(name="accept_1000", op="accept", streams=1000, new_lo=0, new_hi=61),
    ]


def log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "tree", "tree", "score", "accept"])
    if op == "accept":
        return dict(op=op, streams=log_int(rng, 1, 1000), new_lo=rng.choice([0, 1]), new_hi=log_int(rng, 1, 64))
    if op == "score":
        return dict(op=op, rows=log_int(rng, 1, 512), vocab=log_int(rng, 500, 262144), pad=rng.choice([0, 0, 8, 61]), type=rng.choice(["f32", "f16", "bf16"]),
                    softcap=rng.choice([0.0, 30.0]), top=rng.choice([0, 1, 5, 20, 64]))
    nq, nkv, dim = rng.choice([(16, 8, 256), (16, 8, 256), (8, 1, 256), (4, 2, 256), (32, 8, 128), (6, 2, 128), (16, 4, 64), (5, 1, 64)])
    streams = log_int(rng, 1, 64)
    case = dict(op=op, streams=streams, new_lo=rng.choice([0, 1]), new_hi=log_int(rng, 1, 64 if op == "tree" else 16384), prefix=rng.choice([0, 0, 1]) * log_int(rng, 1, 8192),
                old_lo=0, old_hi=rng.choice([0, 1, 1]) * log_int(rng, 1, 8192), nq=nq, nkv=nkv, dim=dim, page=rng.choice([16, 32, 64]),
                window=rng.choice([0, 0, 1]) * log_int(rng, 1, 2048), type=rng.choice(["f16", "bf16"]), pad=rng.choice([0, 0, 7, 64]))
    # no more than the largest listed ones: the products of one 16K prompt, and twice the caches of 64 streams
    while streams * case["new_hi"] * (case["prefix"] + case["old_hi"] + case["new_hi"]) * nq > 1 << 32:
        case["new_hi"] = max(1, case["new_hi"] * 2 // 3)
        case["old_hi"] = case["old_hi"] * 2 // 3
    return case


def ragged(lo, hi, n):
    """n lengths spread evenly over [lo, hi]; a case has the same ones for every seed."""
    return [lo + int((hi - lo) * (i + 0.5) / n + 0.5) for i in range(n)]


def lengths(case):
    """New and cached tokens of each stream, long prompts not always behind long caches."""
    n = case["streams"]
    old = ragged(case.get("old_lo", 0), case.get("old_hi", 0), n)
    return ragged(case["new_lo"], case["new_hi"], n), [old[i * 29 % n] if n % 29 else old[i] for i in range(n)]


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def starts_of(new):
    return ints([0] + torch.tensor(new).cumsum(0).tolist())


def random_trees(new, g):
    """Parents of packed trees: node 0 of each is its root, the others hang from one of the four before them."""
    i = torch.cat([torch.arange(n, device=DEV) for n in new])
    back = 1 + (torch.rand(len(i), generator=g, device=DEV) * i.clamp(max=4)).int().clamp(max=3)
    return torch.where(i > 0, i - back.clamp(max=i), -1).int()


def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(int(seed))
    s = dict(case)
    if case["op"] == "score":
        n, vocab = case["rows"], case["vocab"]
        # a broad body and a few dozen likely tokens per row, mostly among them the given ones
        x = 2.0 * torch.randn(n, vocab + case["pad"], generator=g, device=DEV)
        likely = torch.randint(0, vocab, (n, 48), generator=g, device=DEV)
        x.scatter_add_(1, likely, 12.0 * torch.rand(n, 48, generator=g, device=DEV).sqrt() + 2.0)
        s["logits"] = x.to(TYPES[case["type"]])[:, :vocab]
        anywhere = torch.randint(0, vocab, (n,), generator=g, device=DEV)
        s["targets"] = torch.where(torch.rand(n, generator=g, device=DEV) < 0.7, likely[:, 0], anywhere).int()
        return s
    new, old = lengths(case)
    order = torch.randperm(len(new), generator=torch.Generator().manual_seed(int(seed))).tolist()
    new, old = [new[i] for i in order], [old[i] for i in order]
    s["new"], s["old"], s["starts"] = new, old, starts_of(new)
    total = sum(new)
    if case["op"] in ("tree", "accept"):
        s["parents"] = random_trees(new, g)
    if case["op"] == "accept":
        # sampled tokens that often are what was drafted
        s["sampled"] = torch.randint(0, 262144, (total,), generator=g, device=DEV).int()
        first = torch.repeat_interleave(s["starts"][:-1].long(), ints(new).long())
        wild = torch.randint(0, 262144, (total,), generator=g, device=DEV).int()
        hit = (torch.rand(total, generator=g, device=DEV) < 0.6) & (s["parents"] >= 0)
        s["drafted"] = torch.where(hit, s["sampled"][(first + s["parents"]).clamp(min=0)], wild)
        return s
    t, nq, nkv, dim, page, rows = TYPES[case["type"]], case["nq"], case["nkv"], case["dim"], case["page"], total + case["pad"]
    # q, k and v as a program has them: slices of the fused q|k|v activations; scores with a
    # spread of about 2.5, as normalised heads have
    qkv = torch.randn(rows, nq + 2 * nkv, dim, generator=g, device=DEV)
    qkv[:, :nq] *= 2.5
    qkv = qkv.to(t)
    s["q"], s["k"], s["v"] = qkv[:, :nq], qkv[:, nq:nq + nkv], qkv[:, nq + nkv:]
    if case["pad"]:
        s["out"] = torch.randn(rows, nq, dim, generator=g, device=DEV).to(t)
    s["scale"] = dim ** -0.5
    if not case["prefix"] and not max(old):
        return s
    # pages anywhere in the pool
    shared, need = (case["prefix"] + page - 1) // page, [(n + page - 1) // page for n in old]
    pages = shared + sum(need) + 8
    s["k_pool"] = torch.randn(pages, page, nkv, dim, generator=g, device=DEV).to(t)
    s["v_pool"] = torch.randn(pages, page, nkv, dim, generator=g, device=DEV).to(t)
    free = torch.randperm(pages, generator=g, device=DEV).int()
    s["prefix_table"], free = free[:shared].contiguous(), free[shared:]
    need = ints(need).long()
    column = torch.arange(max(1, int(need.max())), device=DEV)
    at = (torch.cumsum(need, 0) - need)[:, None] + column
    s["table"] = torch.where(column < need[:, None], free[at.clamp(max=len(free) - 1)], -1).int()
    s["lens"] = ints(old)
    return s


# ---- plain forms ---------------------------------------------------------------


def attend(q, k, v, seen, scale):
    """softmax(scale q k^T) v over the keys that each query sees; zeros where it sees none.
    q [..., tokens, nq, dim], k and v [..., keys, nkv, dim], seen [..., tokens, keys]."""
    *lead, n, nq, dim = q.shape
    nkv = k.shape[-2]
    q = q.float().view(*lead, n, nkv, nq // nkv, dim) * scale
    scores = torch.einsum("...nhgd,...khd->...hgnk", q, k.float())
    scores.masked_fill_(~seen[..., None, None, :, :], -math.inf)
    scores.sub_(scores.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    total = scores.sum(-1).clamp(min=1e-30)
    o = torch.einsum("...hgnk,...khd->...nhgd", scores, v.float())
    return (o / total.movedim(-1, -3)[..., None]).reshape(*lead, n, nq, dim)


def cached(s, pool, b=None):
    """The shared prefix's rows and the stream's own cached ones (b None: of all streams, to the table's width)."""
    page, (nkv, dim) = s["page"], s[pool].shape[2:]
    rows = s[pool].view(-1, nkv, dim)
    i = torch.arange(s["prefix"], device=DEV)
    shared = rows[s["prefix_table"][i // page].long() * page + i % page]
    i = torch.arange(s["old"][b] if b is not None else s["table"].shape[1] * page, device=DEV)
    if b is not None:
        return torch.cat([shared, rows[s["table"][b, i // page].long() * page + i % page]])
    mine = rows[s["table"][:, i // page].clamp(min=0).long() * page + i % page]
    return torch.cat([shared.expand(len(mine), -1, -1, -1), mine], 1)


def plain_prompt(s):
    out = s["out"] if s["pad"] else torch.empty_like(s["q"])
    begin = 0
    for b, n in enumerate(s["new"]):  # sequences of very different lengths: one at a time, none padded
        if not n:
            continue
        rows = slice(begin, begin + n)
        begin += n
        before = s["prefix"] + s["old"][b]
        k, v = s["k"][rows], s["v"][rows]
        if "k_pool" in s:
            k, v = torch.cat([cached(s, "k_pool", b), k]), torch.cat([cached(s, "v_pool", b), v])
        at, key = torch.arange(before, before + n, device=DEV)[:, None], torch.arange(before + n, device=DEV)
        seen = key <= at
        if s["window"]:
            seen &= key > at - s["window"]
        out[rows] = attend(s["q"][rows], k, v, seen, s["scale"]).to(out.dtype)
    return out


def ancestors(parents, row, i, streams, most):
    """[streams, most, most]: whether node j lies on node i's path to its root, itself among it."""
    up = torch.zeros(streams, most, most, device=DEV)
    child = parents >= 0
    up[row[child], i[child], parents[child].long()] = 1
    up += torch.eye(most, device=DEV)
    for _ in range(max(1, most - 1).bit_length()):
        up = (up @ up).clamp(max=1)
    return up


def packed(s):
    """Stream and node of every packed row, and the largest number of nodes."""
    new = s["starts"][1:] - s["starts"][:-1]
    row = torch.repeat_interleave(torch.arange(len(new), device=DEV), new.long())
    return row, torch.arange(len(row), device=DEV) - s["starts"][row], max(s["new"])


def plain_tree(s):
    row, i, most = packed(s)
    n, prefix = s["streams"], s["prefix"]
    here = len(row)

    def padded(x):
        y = x.new_zeros(n, most, *x.shape[1:])
        y[row, i] = x[:here]
        return y

    up = ancestors(s["parents"], row, i, n, most)
    depth = up.sum(-1) - 1
    k, v, seen = padded(s["k"]), padded(s["v"]), up > 0
    own_at = (prefix + torch.tensor(s["old"], device=DEV))[:, None] + depth  # positions of the nodes
    key_at = own_at
    if "k_pool" in s:
        k, v = torch.cat([cached(s, "k_pool"), k], 1), torch.cat([cached(s, "v_pool"), v], 1)
        width = s["table"].shape[1] * s["page"]
        j = torch.arange(prefix + width, device=DEV)
        there = j < prefix + s["lens"][:, None]
        seen = torch.cat([there[:, None].expand(-1, most, -1), seen], 2)
        key_at = torch.cat([j.expand(n, -1), own_at], 1)
    if s["window"]:
        seen = seen & (key_at[:, None] > own_at[:, :, None] - s["window"])
    o = attend(padded(s["q"]), k, v, seen, s["scale"])[row, i].to(s["q"].dtype)
    if not s["pad"]:
        return o
    s["out"][:here] = o
    return s["out"]


def plain_score(s):
    x = s["logits"].float()
    n, vocab = x.shape
    lowest = torch.finfo(s["logits"].dtype).min
    x = torch.where(torch.isnan(x) | (x <= lowest), -math.inf, x)
    target = s["targets"].long()[:, None]
    given = x.gather(1, target)
    ranks = 1 + ((x > given) | ((x == given) & (torch.arange(vocab, device=DEV) < target))).sum(1)
    top, ids = torch.sort(x, dim=1, descending=True, stable=True)
    top, ids = top[:, :s["top"]], ids[:, :s["top"]]

    def capped(y):
        return torch.tanh(y / s["softcap"]) * s["softcap"] if s["softcap"] else y

    hidden = x == -math.inf
    x = torch.where(hidden, -math.inf, capped(x))
    x = x - x.amax(1, keepdim=True)
    e = torch.exp(x)
    # the sums in 64 bits: 262,144 terms, and an entropy that is a difference
    total = e.sum(1, dtype=torch.float64)
    log_total = torch.log(total)
    entropy = log_total - torch.where(hidden, 0.0, x * e).sum(1, dtype=torch.float64) / total
    highest = capped(torch.where(hidden, -math.inf, s["logits"].float()).amax(1, keepdim=True))
    return dict(logprobs=(x.gather(1, target)[:, 0].double() - log_total).float(), entropy=entropy.float(), ranks=ranks.int(), top_ids=ids.int(),
                top_logprobs=((capped(top) - highest).double() - log_total[:, None]).float())


def plain_accept(s):
    row, i, most = packed(s)
    n, total = s["streams"], len(row)
    first = s["starts"][row].long()
    up = ancestors(s["parents"], row, i, n, most)
    # a node agrees where its token is its parent's sampled one and no earlier sibling's is
    parent = first + s["parents"].clamp(min=0)
    agrees = (s["parents"] >= 0) & (s["drafted"] == s["sampled"][parent])
    by_parent = torch.full((total,), most, device=DEV).scatter_reduce(0, parent, torch.where(agrees, i, most), "amin")
    agrees &= i == by_parent[parent]
    agrees |= i == 0
    off = torch.zeros(n, most, device=DEV)
    off[row, i] = (~agrees).float()
    kept = torch.einsum("nij,nj->ni", up, off)[row, i] == 0
    counts = torch.zeros(n, dtype=torch.long, device=DEV).scatter_add(0, row, kept.long())
    last = torch.full((n,), -1, device=DEV).scatter_reduce(0, row, torch.where(kept, torch.arange(total, device=DEV), -1), "amax")
    after = torch.where(last >= 0, s["sampled"][last.clamp(min=0)], -1)
    place = torch.cumsum(kept, 0) - 1
    return dict(counts=counts.int(), next=after.int(), kept=torch.where(kept, place, -1).int())


def run(state):
    s = state
    if not own:
        return {"prompt": plain_prompt, "tree": plain_tree, "score": plain_score, "accept": plain_accept}[s["op"]](s)
    if s["op"] == "score":
        from channel_b200 import sampling
        r = sampling.score_rows(s["logits"], s["targets"], top=s["top"], softcap=s["softcap"])
        return dict(logprobs=r.logprobs, entropy=r.entropy, ranks=r.ranks, top_ids=r.top_ids, top_logprobs=r.top_logprobs)
    if s["op"] == "accept":
        from channel_b200 import sampling
        r = sampling.accept_drafts(s["drafted"], s["parents"], s["starts"], s["sampled"])
        return dict(counts=r.counts, next=r.next_tokens, kept=r.kept)
    from channel_b200 import paged
    more = dict(window=s["window"], scale=s["scale"], out=s.get("out"))
    if "k_pool" in s:
        more.update(k_pool=s["k_pool"], v_pool=s["v_pool"], table=s["table"], lens=s["lens"], prefix_table=s["prefix_table"], prefix_len=s["prefix"])
    if s["op"] == "tree":
        return paged.tree_attention(s["q"], s["k"], s["v"], s["starts"], s["parents"], **more)
    return paged.prompt_attention(s["q"], s["k"], s["v"], s["starts"], **more)


# ---- what a pass cannot do without ------------------------------------------------


def work(case):
    if case["op"] == "score":
        return dict(bytes=case["rows"] * (case["vocab"] * SIZE[case["type"]] + 16 + 8 * case["top"]), flops=0)
    new, old = lengths(case)
    if case["op"] == "accept":
        return dict(bytes=4 * (4 * sum(new) + 3 * len(new)) + 4, flops=0)
    prefix, window = case["prefix"], case["window"] or 1 << 40
    pairs, cache_rows, deepest = 0, 0, 0
    for n, length in zip(new, old):
        before = prefix + length
        if not n:
            continue
        if case["op"] == "prompt":
            whole = min(n, max(0, window - before))  # tokens that see all in front of them
            pairs += whole * before + whole * (whole + 1) // 2 + (n - whole) * window
        else:  # a node of a random tree: its cache, and a path of about log2 of its number
            pairs += sum(min(window, before + 1 + int(math.log2(i + 1))) for i in range(n))
        low = max(0, before + 1 - window)  # what the first token sees
        cache_rows += length - max(0, low - prefix) if low < before else 0
        deepest = max(deepest, prefix - low)
    cache_rows += max(0, deepest)
    row = case["dim"] * SIZE[case["type"]]
    bytes_ = 2 * cache_rows * case["nkv"] * row + 2 * sum(new) * (case["nq"] + case["nkv"]) * row + 4 * (cache_rows // case["page"] + 2 * len(new))
    return dict(bytes=bytes_ + (4 * sum(new) if case["op"] == "tree" else 0), flops=4 * case["nq"] * case["dim"] * pairs)


# ---- the definitions in 64 bits ------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "accept":
        return None  # whole numbers only
    if case["op"] == "score":
        x = s["logits"].double()
        x = torch.where(torch.isnan(x) | (x <= torch.finfo(s["logits"].dtype).min), -math.inf, x)
        order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :s["top"]]
        if s["softcap"]:
            x = torch.where(x == -math.inf, x, s["softcap"] * torch.tanh(x / s["softcap"]))
        x = torch.log_softmax(x, 1)
        entropy = -torch.where(x == -math.inf, 0.0, x.exp() * x).sum(1)
        return dict(logprobs=x.gather(1, s["targets"].long()[:, None])[:, 0], entropy=entropy, ranks=None, top_ids=None, top_logprobs=x.gather(1, order))
    group, page = s["nq"] // s["nkv"], case["page"]
    out = s["out"].double() if case["pad"] else torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    parents = s["parents"].tolist() if case["op"] == "tree" else None
    begin = 0
    for b, n in enumerate(s["new"]):
        if not n:
            continue
        k, v = s["k"][begin:begin + n], s["v"][begin:begin + n]
        if "k_pool" in s:
            for own_table, count in ((s["table"][b], s["old"][b]), (s["prefix_table"], case["prefix"])):
                used = own_table[:(count + page - 1) // page].long()
                k = torch.cat([s["k_pool"][used].flatten(0, 1)[:count], k])
                v = torch.cat([s["v_pool"][used].flatten(0, 1)[:count], v])
        before = len(k) - n
        if parents is None:
            at = list(range(before, before + n))
            own_seen = torch.ones(n, n, dtype=torch.bool, device=DEV).tril()
        else:
            at, lists = [], []
            for i in range(n):
                path, j = [], i
                while j >= 0:
                    path.append(j)
                    j = parents[begin + j]
                at.append(before + len(path) - 1)
                lists.append([float(j in path) for j in range(n)])
            own_seen = torch.tensor(lists, device=DEV) > 0
        at = torch.tensor(at, device=DEV)
        hidden = torch.cat([torch.zeros(n, before, dtype=torch.bool, device=DEV), ~own_seen], 1)
        if case["window"]:
            hidden |= torch.cat([torch.arange(before, device=DEV), at])[None] <= at[:, None] - case["window"]
        for h in range(s["nq"]):
            z = s["q"][begin:begin + n, h].double() @ k[:, h // group].double().T * s["scale"]
            out[begin:begin + n, h] = torch.softmax(z.masked_fill(hidden, -math.inf), 1) @ v[:, h // group].double()
        begin += n
    return out
