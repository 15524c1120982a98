"""A paged KV cache of limited size: decode over a prefix that a batch shares, attention that adds up what each cached token weighs, and the
eviction of tokens that weigh least - as cases that can be timed and compared.

Pools are [blocks, block_size, kv_heads, D], a sequence's tokens lie in the pages of its row of the page table. With scale = 1 / sqrt(D) and
G = heads / kv_heads query heads to a kv head,
    p[i, h, j] = exp(scale * q[i, h] . k[j]) / (sum over the keys visible to token i),   out[i, h] = sum over j of p[i, h, j] * v[j],
    weights[s, g, j] += sum over the call's tokens i of sequence s and the query heads h of kv head g of p[i, h, j].
Eviction works on each kv head of each sequence alone. Of n tokens, where n > m = max(keep, first + recent), it keeps the first `first`, the last
`recent`, and of those in between the m - first - recent of the largest weights (equal ones: the lower index). Afterwards the sequence has m:
[0, first) and [m - recent, m) hold the first and the last in order; in [first, m - recent) those kept stay where they are, and the i-th place
that has come free takes the i-th of those kept behind m - recent, both counted upwards. weights go along, what lies behind them is 0.

Kinds of case (field "kind"):
  weigh   one token per sequence against its pages, weights added up
  prompt  new tokens of every sequence (already in the cache) against all of it, causal; weights of all new tokens or of the last ones
  shared  one token per sequence; the sequences of a group have the pages of a prefix in common. Where "weights" is true, the weights of the
          tokens behind those pages are added up
  evict   the cache of a batch is brought down to m tokens a sequence

`own` says who computes: False the plain form below, elementary torch operations in 32 bits; True the operators of scicompute_attention_b200.ops.
Lengths of ragged batches are spread evenly over a case's range and dealt to the sequences in an order made from the seed. Keys and values have
channels of different sizes, as projections give them; the pool's other slots hold what earlier sequences left there.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}

# No drawn case does more than the largest listed ones, nor makes scores that the plain form cannot hold.
MOST_FLOPS = 1.28e11
MOST_BYTES = 2.5e9
MOST_SCORES = 1.6e9


def listed():
    layer = {"heads": 32, "kv_heads": 8, "head_dim": 128, "dtype": "bf16", "block_size": 16}
    return [
        # one user, a short context: the latency of a step
        dict(layer, name="weigh_one_sequence", kind="weigh", seqs=1, min_len=701, max_len=701),
        # a server that keeps the weights of 192 conversations
        dict(layer, name="weigh_192_sequences", kind="weigh", seqs=192, min_len=500, max_len=6000),
        # small heads of which sixteen share a kv head, larger pages
        dict(layer, name="weigh_d64_sixteen_heads_to_one", kind="weigh", kv_heads=2, head_dim=64, dtype="fp16", block_size=32, seqs=96, min_len=200,
             max_len=6001),
        # a short follow-up of one conversation
        dict(layer, name="prompt_one_short", kind="prompt", seqs=1, min_new=37, max_new=37, min_len=733, max_len=733, last=0),
        # whole prompts enter the cache, every token of theirs is weighed: bound by the tensor cores
        dict(layer, name="prompt_four_whole", kind="prompt", seqs=4, min_new=1900, max_new=2048, min_len=1900, max_len=2048, last=0),
        # long follow-up prompts of which the last 64 tokens say what is worth keeping; small heads, fp16
        dict(layer, name="prompt_d64_last_tokens", kind="prompt", head_dim=64, dtype="fp16", block_size=32, seqs=9, min_new=100, max_new=900,
             min_len=1000, max_len=3500, last=64),
        # five answers to one question: latency
        dict(layer, name="shared_five_answers", kind="shared", groups=1, min_group=5, max_group=5, min_prefix=501, max_prefix=501, min_len=1,
             max_len=200, weights=False),
        # 128 conversations behind one system prompt of 8 thousand tokens
        dict(layer, name="shared_system_prompt", kind="shared", groups=1, min_group=128, max_group=128, min_prefix=8101, max_prefix=8101, min_len=20,
             max_len=1500, weights=False),
        # sampled continuations, 4 to 12 of each of 14 prompts, whose own tokens are weighed
        dict(layer, name="shared_continuations_weights", kind="shared", dtype="fp16", groups=14, min_group=4, max_group=12, min_prefix=300,
             max_prefix=4000, min_len=1, max_len=700, weights=True),
        # one conversation, a little over its budget: latency
        dict(layer, name="evict_one_sequence", kind="evict", seqs=1, min_len=1100, max_len=1100, keep=1024, recent=64, first=4),
        # one document of 100 thousand tokens is brought down to 8 thousand
        dict(layer, name="evict_long_document", kind="evict", seqs=1, min_len=100003, max_len=100003, keep=8000, recent=500, first=4),
        # the cache of a full server is brought down to two thousand tokens a conversation
        dict(layer, name="evict_192_sequences", kind="evict", seqs=192, min_len=500, max_len=6000, keep=2000, recent=250, first=4),
    ]


# ------------------------------------------------------------------------------------------------
# drawn cases
# ------------------------------------------------------------------------------------------------
def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        case = _draw(rng)
        w = work(case)
        if w["flops"] > MOST_FLOPS or w["bytes"] > MOST_BYTES:
            continue
        if case["kind"] == "evict":
            if case["max_len"] > _limit(case):  # otherwise nothing is evicted
                return case
            continue
        rows, longest = len(_lengths(case)), max(n for _, n in _lengths(case))
        if rows * longest * case["heads"] * case.get("max_new", 1) <= MOST_SCORES and rows * longest * case["kv_heads"] * case["head_dim"] <= 2.5e9:
            return case


def _draw(rng):
    heads, kv_heads = rng.choice([(32, 8), (32, 8), (32, 8), (8, 8), (16, 2), (6, 3), (32, 2)])
    case = {"heads": heads, "kv_heads": kv_heads, "head_dim": rng.choice([64, 96, 128, 128, 128, 256]),
            "dtype": rng.choice(["bf16", "bf16", "fp16"]), "block_size": rng.choice([8, 16, 16, 16, 32, 64])}
    kind = rng.choice(["weigh", "prompt", "shared", "evict"])
    if kind == "weigh":
        lo = _log(rng, 1, 1500)
        return dict(case, kind=kind, seqs=_log(rng, 1, 256), min_len=lo, max_len=lo + _log(rng, 1, 20000))
    if kind == "prompt":
        new, lo = _log(rng, 1, 1000), _log(rng, 1, 2000)
        most_new = new + _log(rng, 1, 1000)
        return dict(case, kind=kind, seqs=_log(rng, 1, 32), min_new=new, max_new=most_new, min_len=lo + most_new,
                    max_len=lo + most_new + _log(rng, 1, 8000), last=rng.choice([0, 0, 0, 1, 32, 64]))
    if kind == "shared":
        group, prefix, lo = _log(rng, 1, 200), _log(rng, 1, 8000), _log(rng, 1, 800)
        return dict(case, kind=kind, groups=_log(rng, 1, 20), min_group=group, max_group=group + _log(rng, 1, 20), min_prefix=prefix,
                    max_prefix=prefix + _log(rng, 1, 4000), min_len=lo, max_len=lo + _log(rng, 1, 1500), weights=rng.random() < 0.4)
    lo = _log(rng, 1, 4000)
    keep = _log(rng, 8, 8000)
    return dict(case, kind=kind, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), seqs=_log(rng, 1, 256), min_len=lo, max_len=lo + _log(rng, 1, 30000),
                keep=keep, recent=rng.randint(0, keep // 2), first=rng.choice([0, 1, 4, 4, keep // 4]))


# ------------------------------------------------------------------------------------------------
# sizes that follow from a case
# ------------------------------------------------------------------------------------------------
def _spread(lo, hi, n):
    """n whole lengths, evenly over [lo, hi]."""
    return [(lo + hi) // 2] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _groups(case):
    """(sequences, tokens of the prefix) of every group."""
    return list(zip(_spread(case["min_group"], case["max_group"], case["groups"]), _spread(case["min_prefix"], case["max_prefix"], case["groups"])[::-1]))


def _lengths(case):
    """(new tokens, tokens in the cache with them) of every sequence; of a "shared" case without the prefix's."""
    if case["kind"] == "shared":
        return [(1, n) for n in _spread(case["min_len"], case["max_len"], sum(n for n, _ in _groups(case)))]
    total = _spread(case["min_len"], case["max_len"], case["seqs"])
    if case["kind"] == "prompt":
        return list(zip(_spread(case["min_new"], case["max_new"], case["seqs"]), total))
    return [(1, n) for n in total]


def _limit(case):
    return max(case["keep"], case["first"] + case["recent"])


def work(case):
    """Bytes: every input read once, every output written once; a shared prefix counts once. FLOPs: 4 * D for every visible (query, key) pair.
    Eviction: the weights of what is over its limit, read and written, and the rows that move - the last ones, and those in places that come free
    if every token in between is kept with the same probability."""
    hq, hkv, d, e, bs = case["heads"], case["kv_heads"], case["head_dim"], BYTES[case["dtype"]], case["block_size"]
    lens = _lengths(case)
    if case["kind"] == "evict":
        m, rows, weights = _limit(case), 0.0, 0
        for _, n in lens:
            if n > m:
                stay, between = m - case["first"] - case["recent"], n - case["first"] - case["recent"]
                rows += case["recent"] + stay * (1 - stay / between)
                weights += n
        return {"bytes": int(hkv * (4 * rows * d * e + 8 * weights)) + 8 * len(lens), "flops": 0}
    new = sum(q for q, _ in lens)
    flops, tokens, weighed, blocks = 0, sum(n for _, n in lens), 0, sum(-(-n // bs) for _, n in lens)
    if case["kind"] == "shared":
        groups = _groups(case)
        flops = 4 * hq * d * (tokens + sum(n * p for n, p in groups))
        weighed = sum(n * (p % bs) for n, p in groups) + tokens if case["weights"] else 0
        tokens += sum(p // bs * bs + n * (p % bs) for n, p in groups)
    else:
        flops = 4 * hq * d * sum(q * n - q * (q - 1) // 2 for q, n in lens)
        weighed = tokens
    return {"bytes": 2 * tokens * hkv * d * e + 2 * new * hq * d * e + 8 * weighed * hkv + 4 * blocks + 4 * len(lens), "flops": flops}


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _pool(gen, case, blocks, channels):
    """Rows of K or V in every slot."""
    pool = torch.empty((blocks, case["block_size"]) + channels.shape, dtype=DTYPES[case["dtype"]], device="cuda")
    piece = max(1, (1 << 27) // (case["block_size"] * channels.numel()))
    for at in range(0, blocks, piece):
        part = pool[at:at + piece]
        part.copy_(torch.randn(part.shape, generator=gen, device="cuda") * channels)
    return pool


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    order = np.random.default_rng(seed)
    hq, hkv, d, bs = case["heads"], case["kv_heads"], case["head_dim"], case["block_size"]
    lens = _lengths(case)
    lens = [lens[i] for i in order.permutation(len(lens))]
    new, keys = np.array([q for q, _ in lens]), np.array([n for _, n in lens])
    seqs = len(lens)
    shared = np.zeros(seqs, dtype=np.int64)  # blocks that a sequence has in common with the one before it
    s = {"case": case}
    prefix_blocks = np.zeros(seqs, dtype=np.int64)
    if case["kind"] == "shared":
        groups = _groups(case)
        s["cu_groups"] = np.concatenate([[0], np.cumsum([n for n, _ in groups])]).astype(np.int32)
        s["prefix_lens"] = np.array([p for _, p in groups], dtype=np.int32)
        for (first, end), (_, p) in zip(zip(s["cu_groups"], s["cu_groups"][1:]), groups):
            keys[first:end] += p
            prefix_blocks[first:end] = p // bs
            shared[first + 1:end] = p // bs
    counts = -(-keys // bs)
    taken = counts - shared
    blocks = int(taken.sum() + taken.sum() // 8 + 16)  # the pool is never quite full
    k_channels, v_channels = (torch.exp(0.5 * torch.randn((hkv, d), generator=gen, device="cuda")) for _ in range(2))
    s["k"], s["v"] = _pool(gen, case, blocks, k_channels), _pool(gen, case, blocks, v_channels)

    # page table [sequences, pages of the longest there may be]: blocks dealt from a shuffled pool; -1 behind a sequence's last block
    ids = order.permutation(blocks).astype(np.int32)
    table = np.full((seqs, -(-(case["max_len"] + case.get("max_prefix", 0)) // bs)), -1, dtype=np.int32)
    at = 0
    for i in range(seqs):
        table[i, :shared[i]] = table[i - 1, :shared[i]]
        table[i, shared[i]:counts[i]] = ids[at:at + taken[i]]
        at += taken[i]
    s["table"] = torch.from_numpy(table).cuda()
    s["lens"] = torch.from_numpy(keys.astype(np.int32)).cuda()
    pos = torch.arange(table.shape[1] * bs, device="cuda")
    if case.get("weights", True):
        # what earlier steps have left: heavy and light tokens, some that nobody has looked at, 0 behind the last
        w = torch.exp(1.5 * torch.randn((seqs, hkv, pos.numel()), generator=gen, device="cuda") - 2)
        w *= torch.rand(w.shape, generator=gen, device="cuda") > 0.02
        s["weights"] = w * (pos < s["lens"][:, None, None])
    if case["kind"] == "evict":
        return s
    s["mean"], s["longest"] = int(keys.sum()) // seqs, int(keys.max())
    q = torch.randn((int(new.sum()), hq, d), generator=gen, device="cuda").to(DTYPES[case["dtype"]])
    if case["kind"] == "prompt":
        s["q"] = q
        s["cu"], s["host_lens"] = np.concatenate([[0], np.cumsum(new)]).astype(np.int32), keys.astype(np.int32)
    else:
        s["q"] = q.view(seqs, hq, 1, d)
    if case["kind"] == "shared":
        s["own_from"] = torch.from_numpy(prefix_blocks * bs).cuda()  # the first token behind the common pages
    return s


# ------------------------------------------------------------------------------------------------
# the plain form
# ------------------------------------------------------------------------------------------------
def _attention(q, s, visible, counted):
    """q [sequences, rows, heads, D] over the sequences' pages; visible [sequences, rows, keys]. Output, and the weights of the rows where
    counted [sequences, rows] holds, [sequences, kv_heads, keys]."""
    n, rows, hq, d = q.shape
    hkv = s["case"]["kv_heads"]
    ids = s["table"].long().clamp(min=0)
    q = q.float().view(n, rows, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(n, hkv, -1, d)
    k = s["k"][ids].float().view(n, -1, hkv, d)
    scores = torch.matmul(q, k.permute(0, 2, 3, 1)).mul_(1.0 / math.sqrt(d))
    del k
    scores = scores.view(n, hkv, hq // hkv, rows, -1)
    scores.masked_fill_(~visible[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(top > -math.inf, top, 0.0)).exp_()
    total = scores.sum(-1, keepdim=True)
    scores.mul_(torch.where(total > 0, 1.0 / total, 0.0))
    v = s["v"][ids].float().view(n, -1, hkv, d)
    out = torch.matmul(scores.view(n, hkv, (hq // hkv) * rows, -1), v.transpose(1, 2)).view(n, hkv, hq // hkv, rows, d)
    del v
    share = scores.mul_(counted[:, None, None, :, None]).sum((2, 3))
    return out.permute(0, 3, 1, 2, 4).reshape(n, rows, hq, d), share


def _plain_evict(s):
    case = s["case"]
    k, v, bs, hkv = s["k"], s["v"], case["block_size"], case["kv_heads"]
    first, recent, m = case["first"], case["recent"], _limit(case)
    w = s["weights"].clone()
    lens = s["lens"].long()
    new_lens = lens.clamp(max=m)
    over = torch.nonzero(lens > m)[:, 0]
    stay = m - first - recent
    for part in over.split(max(1, (1 << 25) // (hkv * w.shape[2]))):
        n = lens[part][:, None, None]
        pos = torch.arange(w.shape[2], device="cuda").expand(part.numel(), hkv, -1)
        # the tokens in between, heaviest first; a stable sort leaves equal ones in their order
        between = (pos >= first) & (pos < n - recent)
        rank = torch.sort(torch.where(between, w[part], -1.0), dim=-1, descending=True, stable=True).indices
        kept = torch.zeros_like(between)
        kept.scatter_(2, rank[..., :stay], True)
        free = between & ~kept & (pos < m - recent)
        moves = kept & (pos >= m - recent)
        # the i-th free place takes the i-th token that moves
        row_to, at_to = torch.nonzero(free.view(-1, pos.shape[2]), as_tuple=True)
        row_from, at_from = torch.nonzero(moves.view(-1, pos.shape[2]), as_tuple=True)
        tail = torch.arange(recent, device="cuda").expand(part.numel() * hkv, -1).reshape(-1)
        row_tail = torch.arange(part.numel() * hkv, device="cuda")[:, None].expand(-1, recent).reshape(-1)
        row = torch.cat([row_to, row_tail])
        seq, head = part[row // hkv], row % hkv
        src = torch.cat([at_from, lens[seq[row_to.numel():]] - recent + tail])
        dst = torch.cat([at_to, m - recent + tail])
        block_from, block_to = s["table"][seq, src // bs].long(), s["table"][seq, dst // bs].long()
        for pool in (k, v):
            pool[block_to, dst % bs, head] = pool[block_from, src % bs, head]
        moved = w[seq, head, src]
        w[seq, head, dst] = moved
        w[part] = torch.where(pos < m, w[part], 0.0)
    return [k, v, w, new_lens.to(torch.int32)]


def _plain(s):
    case = s["case"]
    if case["kind"] == "evict":
        return _plain_evict(s)
    dtype, bs = DTYPES[case["dtype"]], case["block_size"]
    pos = torch.arange(s["table"].shape[1] * bs, device="cuda")
    visible = (pos < s["lens"][:, None]) & (s["table"] >= 0).repeat_interleave(bs, 1)
    if case["kind"] != "prompt":
        out, share = _attention(s["q"].transpose(1, 2), s, visible[:, None], torch.ones_like(s["lens"][:, None], dtype=torch.float32))
        out = out.to(dtype).transpose(1, 2)
        if case["kind"] == "shared":
            if not case["weights"]:
                return out
            share = share * (pos >= s["own_from"][:, None, None])
        return [out, s["weights"].add_(share)]
    cu, lens = (torch.from_numpy(x).long().cuda() for x in (s["cu"], s["host_lens"]))
    new = cu[1:] - cu[:-1]
    row = torch.arange(case["max_new"], device="cuda")
    there = row < new[:, None]
    visible = visible[:, None] & there[..., None] & (pos <= (lens - new)[:, None, None] + row[:, None])
    counted = there & (row >= (new - case["last"])[:, None]) if case["last"] else there
    at = (cu[:-1, None] + row).clamp(max=s["q"].shape[0] - 1)
    out, share = _attention(s["q"][at], s, visible, counted.float())
    return [out.to(dtype)[there], s["weights"].add_(share)]


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def run(s):
    """The attention's output and the weights; of an eviction the pools, the weights and the new lengths."""
    if not own:
        return _plain(s)
    from scicompute_attention_b200 import ops
    case = s["case"]
    kind, bs = case["kind"], case["block_size"]
    if kind == "weigh":
        out = ops.paged_attention_weights(s["q"], s["k"], s["v"], s["table"], s["lens"], s["weights"], block_size=bs, typical_len=s["mean"],
                                          longest_len=s["longest"])
        return [out, s["weights"]]
    if kind == "prompt":
        out = ops.flash_attention_paged_weights(s["q"], s["k"], s["v"], s["table"], s["cu"], s["host_lens"], s["weights"], last=case["last"])
        return [out, s["weights"]]
    if kind == "shared":
        out = ops.paged_attention_shared(s["q"], s["k"], s["v"], s["table"], s["lens"], s["cu_groups"], s["prefix_lens"], block_size=bs,
                                         weights=s.get("weights"), typical_len=s["mean"], longest_len=s["longest"])
        return [out, s["weights"]] if case["weights"] else out
    # the weights that decide stay as they are, so that every pass has the same tokens to move
    weights = s["weights"].clone()
    lens = ops.kv_evict(s["k"], s["v"], weights, s["table"], s["lens"], keep=case["keep"], recent=case["recent"], first=case["first"])
    return [s["k"], s["v"], weights, lens]


# ------------------------------------------------------------------------------------------------
# 64 bits
# ------------------------------------------------------------------------------------------------
def _exact_evict(s):
    case = s["case"]
    bs, hkv, first, recent = case["block_size"], case["kv_heads"], case["first"], case["recent"]
    limit = _limit(case)
    pools = [x.clone() for x in (s["k"], s["v"])]
    weights = s["weights"].cpu().numpy().astype(np.float64)
    table, lens = s["table"].cpu().numpy().astype(np.int64), s["lens"].cpu().numpy()
    to, come = [], []  # (block, place in it, head) of every row that moves
    for i, n in enumerate(lens):
        if n <= limit:
            continue
        for h in range(hkv):
            w = weights[i, h]
            middle = np.arange(first, n - recent)
            stay = limit - first - recent
            chosen = np.sort(middle[np.lexsort((middle, -w[middle]))[:stay]])  # by weight, then by index
            places = np.setdiff1d(np.arange(first, limit - recent), chosen, assume_unique=True)
            late = chosen[chosen >= limit - recent]
            dst = np.concatenate([places, np.arange(limit - recent, limit)])
            src = np.concatenate([late, np.arange(n - recent, n)])
            w[dst] = w[src]
            w[limit:] = 0
            to.append((table[i, dst // bs], dst % bs, np.full(dst.size, h)))
            come.append((table[i, src // bs], src % bs, np.full(src.size, h)))
    if to:
        a, b = (tuple(torch.from_numpy(np.concatenate(x)).cuda() for x in zip(*y)) for y in (to, come))
        for pool, old in zip(pools, (s["k"], s["v"])):
            pool[a] = old[b]
    return [*pools, torch.from_numpy(weights).cuda(), torch.from_numpy(np.minimum(lens, limit)).cuda()]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "evict":
        return _exact_evict(s) if sum(n for _, n in _lengths(case)) * case["kv_heads"] <= 2e7 else None
    bs, hkv, d, group = case["block_size"], case["kv_heads"], case["head_dim"], case["heads"] // case["kv_heads"]
    lens = s["lens"].tolist()
    news = np.diff(s["cu"]).tolist() if case["kind"] == "prompt" else [1] * len(lens)
    flat = s["q"].reshape(-1, case["heads"], d)
    weights = s["weights"].double() if "weights" in s else None
    own_from = s["own_from"].tolist() if case["kind"] == "shared" else None
    outs, first = [], 0
    for i, (n, new) in enumerate(zip(lens, news)):
        blocks = s["table"][i, :-(-n // bs)].long()
        k, v = (s[x][blocks].reshape(-1, hkv, d)[:n].double() for x in ("k", "v"))
        q = flat[first:first + new].double()
        first += new
        scores = torch.einsum("ihgd,jhd->hgij", q.view(new, hkv, group, d), k) / math.sqrt(d)
        hidden = torch.arange(n, device="cuda")[None, :] > torch.arange(n - new, n, device="cuda")[:, None]
        p = torch.softmax(scores.masked_fill_(hidden, -math.inf), -1)
        del scores
        outs.append(torch.einsum("hgij,jhd->ihgd", p, v).reshape(new, -1, d))
        if weights is not None:
            start = own_from[i] if case["kind"] == "shared" else 0
            weights[i, :, start:n] += p[:, :, new - min(new, case.get("last", 0) or new):, start:].sum((1, 2))
    out = torch.cat(outs).view(s["q"].shape)
    return out if weights is None else [out, weights]
