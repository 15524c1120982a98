"""The 8-bit paged KV cache - written, read back, and attended over - as cases that can be timed and compared.

A row of the cache is one token of one kv head: D numbers of 8 bits (e4m3) and one scale, a power of two. With x the row,
    e     = the smallest whole number in [-14, 7] with min(max |x|, 57344) <= 448 * 2^e,
    code  = x * 2^-e, rounded to the nearest e4m3 number (ties to even), at most 448 in size; NaN stays NaN,
    value = code * 2^e.
A pool is a pair: codes, float8_e4m3fn [blocks, block_size, kv_heads, D], and scales, uint8 [blocks, kv_heads, block_size
rounded up to 16], which hold e + 15.

Kinds of case (field "kind"):
  step   one decode step of a paged batch: the new token of every sequence is written, then attention over the cache
  chunk  new tokens of every sequence (a follow-up prompt) are written, then their attention over the cache, causal or not
  cache  a prompt batch is written to the pool, blocks are read back (swap, prefix export)

`own` says who computes: False the plain form below, elementary torch operations in 32 bits; True the operators of
scicompute_attention_b200.ops. Lengths of ragged batches are spread evenly over a case's range and dealt to the sequences
in an order made from the seed. Keys and values have channels of different sizes, as projections give them; the pool's
other slots hold what earlier sequences left there.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
FP8 = torch.float8_e4m3fn

# No drawn case does more than the largest listed ones, nor makes scores that the plain form cannot hold.
MOST_FLOPS = 4.5e11
MOST_BYTES = 2.4e9
MOST_SCORES = 2.2e9


def listed():
    layer = {"heads": 32, "kv_heads": 8, "head_dim": 128, "dtype": "bf16", "block_size": 16}
    return [
        # one user, a short context: the latency of a step
        dict(layer, name="step_one_sequence", kind="step", seqs=1, min_len=701, max_len=701),
        # a handful of short conversations
        dict(layer, name="step_few_sequences", kind="step", seqs=6, min_len=33, max_len=900),
        # a full server: 256 sequences of 512 to 8192 tokens scattered over the pool
        dict(layer, name="step_256_sequences", kind="step", seqs=256, min_len=512, max_len=8192),
        # one document of 100 thousand tokens
        dict(layer, name="step_long_document", kind="step", seqs=1, min_len=100003, max_len=100003, block_size=32),
        # small heads of which sixteen share a kv head, larger pages
        dict(layer, name="step_d64_sixteen_heads_to_one", kind="step", heads=32, kv_heads=2, head_dim=64, dtype="fp16",
             block_size=32, seqs=96, min_len=200, max_len=6001),
        # wide heads
        dict(layer, name="step_d256", kind="step", heads=16, kv_heads=2, head_dim=256, seqs=40, min_len=100, max_len=5000),
        # a short follow-up of one conversation: the whole call is a few microseconds of GPU work
        dict(layer, name="chunk_one_short", kind="chunk", causal=True, seqs=1, min_new=37, max_new=37, min_len=733, max_len=733),
        # follow-up prompts: a few hundred new tokens per sequence against the conversation so far
        dict(layer, name="chunk_follow_up_prompts", kind="chunk", causal=True, seqs=20, min_new=16, max_new=500, min_len=512, max_len=6000),
        # long prompts in chunks of about two thousand tokens: bound by the tensor cores
        dict(layer, name="chunk_long_prompts", kind="chunk", causal=True, seqs=4, min_new=1900, max_new=2048, min_len=5000, max_len=8190),
        # small heads, fp16, every new token sees every key
        dict(layer, name="chunk_d64_bidirectional", kind="chunk", causal=False, head_dim=64, dtype="fp16", block_size=32, seqs=9, min_new=100,
             max_new=900, min_len=1000, max_len=3500),
        # a prompt batch enters the pool, blocks are read back
        dict(layer, name="cache_prompts", kind="cache", seqs=24, min_len=64, max_len=4096, gather=1500),
        # one prompt of a small fp16 model
        dict(layer, name="cache_one_prompt", kind="cache", head_dim=64, dtype="fp16", seqs=1, min_len=203, max_len=203, gather=9),
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
        if case["kind"] == "cache" or case["seqs"] * case["max_len"] * case["heads"] * case.get("max_new", 1) <= MOST_SCORES:
            return case


def _draw(rng):
    heads, kv_heads = rng.choice([(32, 8), (32, 8), (32, 8), (8, 8), (16, 2), (6, 3), (32, 2)])
    case = {"heads": heads, "kv_heads": kv_heads, "head_dim": rng.choice([64, 96, 128, 128, 128, 256]),
            "dtype": rng.choice(["bf16", "bf16", "fp16"]), "block_size": rng.choice([8, 16, 16, 16, 32, 64])}
    kind = rng.choice(["step"] * 4 + ["chunk"] * 4 + ["cache"])
    if kind == "step":
        lo = _log(rng, 1, 1500)
        return dict(case, kind=kind, seqs=_log(rng, 1, 256), min_len=lo, max_len=lo + _log(rng, 1, 20000))
    if kind == "chunk":
        new, lo = _log(rng, 1, 1000), _log(rng, 1, 2000)
        most_new = new + _log(rng, 1, 1000)
        return dict(case, kind=kind, causal=rng.random() < 0.75, seqs=_log(rng, 1, 48), min_new=new, max_new=most_new, min_len=lo + most_new,
                    max_len=lo + most_new + _log(rng, 1, 8000))
    lo = _log(rng, 1, 500)
    return dict(case, kind=kind, dtype=rng.choice(["bf16", "fp16", "fp32"]), seqs=_log(rng, 1, 64), min_len=lo,
                max_len=lo + _log(rng, 1, 6000), gather=_log(rng, 1, 4000))


# ------------------------------------------------------------------------------------------------
# sizes that follow from a case
# ------------------------------------------------------------------------------------------------
def _spread(lo, hi, n):
    """n whole lengths, evenly over [lo, hi]."""
    return [(lo + hi) // 2] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _lengths(case):
    """(new tokens, tokens in the cache with them) of every sequence."""
    total = _spread(case["min_len"], case["max_len"], case["seqs"])
    if case["kind"] == "chunk":
        return list(zip(_spread(case["min_new"], case["max_new"], case["seqs"]), total))
    return [(1 if case["kind"] == "step" else n, n) for n in total]


def work(case):
    """Bytes: every input read once, every output written once; D + 1 bytes for a row of the cache. FLOPs: 4 * D for every
    visible (query, key) pair."""
    hq, hkv, d, e = case["heads"], case["kv_heads"], case["head_dim"], BYTES[case["dtype"]]
    lens = _lengths(case)
    new, keys = sum(q for q, _ in lens), sum(n for _, n in lens)
    written = 2 * new * hkv * (d * e + d + 1)  # K and V come in `dtype` and are stored
    if case["kind"] == "cache":
        return {"bytes": written + 4 * new + 2 * case["gather"] * (case["block_size"] * hkv * (d + 1 + d * e) + 4), "flops": 0}
    blocks = sum(-(-n // case["block_size"]) for _, n in lens)
    nbytes = written + 2 * keys * hkv * (d + 1) + 2 * new * hq * d * e + 4 * blocks + 4 * len(lens) + (4 * new if case["kind"] == "chunk" else 0)
    causal = case.get("causal", True)
    return {"bytes": nbytes, "flops": 4 * hq * d * sum(q * n - (q * (q - 1) // 2 if causal else 0) for q, n in lens)}


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _rows(gen, case, n, channels):
    """n rows of K or V, [n, kv_heads, D]."""
    return (torch.randn((n,) + channels.shape, generator=gen, device="cuda") * channels).to(DTYPES[case["dtype"]])


def _filled_pool(gen, case, blocks, channels):
    bs, hkv, d = case["block_size"], case["kv_heads"], case["head_dim"]
    codes = torch.empty((blocks, bs, hkv, d), dtype=FP8, device="cuda")
    scales = torch.full((blocks, hkv, -(-bs // 16) * 16), 15, dtype=torch.uint8, device="cuda")
    piece = max(1, (1 << 26) // (bs * hkv * d))
    for at in range(0, blocks, piece):
        n = min(piece, blocks - at)
        c, s = _quantise(_rows(gen, case, n * bs, channels))
        codes.view(torch.uint8)[at:at + n] = c.view(torch.uint8).view(n, bs, hkv, d)
        scales[at:at + n, :, :bs] = s.view(n, bs, hkv).transpose(1, 2)
    return codes, scales


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    order = np.random.default_rng(seed)
    hq, hkv, d, bs = case["heads"], case["kv_heads"], case["head_dim"], case["block_size"]
    lens = _lengths(case)
    lens = [lens[i] for i in order.permutation(len(lens))]
    new, keys = [q for q, _ in lens], [n for _, n in lens]
    counts = [-(-n // bs) for n in keys]
    blocks = sum(counts) + sum(counts) // 8 + 16  # the pool is never quite full
    s = {"case": case}
    k_channels, v_channels = (torch.exp(0.5 * torch.randn((hkv, d), generator=gen, device="cuda")) for _ in range(2))
    s["k"], s["v"] = _filled_pool(gen, case, blocks, k_channels), _filled_pool(gen, case, blocks, v_channels)
    s["k_new"], s["v_new"] = _rows(gen, case, sum(new), k_channels), _rows(gen, case, sum(new), v_channels)

    # page table [sequences, longest]: blocks dealt from a shuffled pool; -1 behind a sequence's last block
    ids = torch.randperm(blocks, generator=gen, device="cuda").to(torch.int32)
    n = torch.tensor(counts, device="cuda")
    first = torch.cumsum(n, 0) - n
    col = torch.arange(max(counts), device="cuda")
    at = first[:, None] + col[None, :]
    s["table"] = torch.where(col[None, :] < n[:, None], ids[at.clamp(max=blocks - 1)], torch.full_like(at, -1, dtype=torch.int32)).contiguous()
    s["lens"] = torch.tensor(keys, dtype=torch.int32, device="cuda")  # the new tokens included
    if case["kind"] != "step":
        # slot of every new token: the last ones of its sequence
        seq = torch.repeat_interleave(torch.arange(len(new), device="cuda"), torch.tensor(new, device="cuda"))
        start = torch.tensor(np.concatenate([[0], np.cumsum(new)[:-1]]), device="cuda")
        pos = torch.arange(sum(new), device="cuda") - start[seq] + (s["lens"] - torch.tensor(new, device="cuda"))[seq]
        s["slots"] = (s["table"][seq, pos // bs] * bs + pos % bs).to(torch.int32)
    if case["kind"] == "cache":
        s["gather"] = ids[torch.randperm(blocks, generator=gen, device="cuda")[:case["gather"]]].contiguous()
        if s["gather"].numel() < case["gather"]:  # more blocks than the pool has: some come twice
            s["gather"] = s["gather"][torch.arange(case["gather"], device="cuda") % s["gather"].numel()].contiguous()
        return s
    q = torch.randn((sum(new), hq, d), generator=gen, device="cuda").to(DTYPES[case["dtype"]])
    if case["kind"] == "step":
        s["q"] = q.view(len(new), hq, 1, d)
        s["mean"], s["longest"] = sum(keys) // len(keys), max(keys)
    else:
        s["q"] = q
        s["cu"], s["host_lens"] = np.concatenate([[0], np.cumsum(new)]).astype(np.int32), np.array(keys, dtype=np.int32)
    return s


# ------------------------------------------------------------------------------------------------
# the plain form
# ------------------------------------------------------------------------------------------------
def _power(e):
    """2^e in 32 bits, to the bit: its exponent field, put together."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _quantise(rows):
    """Codes and e + 15 of rows [..., D]."""
    x = rows.float()
    amax = torch.nan_to_num(x.abs(), nan=0.0).amax(-1).clamp(max=57344.0)
    part, exponent = torch.frexp(amax)  # amax = part * 2^exponent, part in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(amax > 0, exponent - 9 + (part > 0.875), -14).clamp(-14, 7)
    codes = torch.clamp(x * _power(-e)[..., None], -448.0, 448.0).to(FP8)
    return codes, (e + 15).to(torch.uint8)


def _store(pool, slots, rows):
    codes, scales = pool
    bs = codes.shape[1]
    c, e = _quantise(rows)
    slots = slots.long()
    codes.view(torch.uint8).view((-1,) + codes.shape[2:])[slots] = c.view(torch.uint8)
    scales.transpose(1, 2)[slots // bs, slots % bs] = e


def _read(pool, ids):
    """Values of the blocks `ids`, [*ids.shape, block_size, kv_heads, D], in 32 bits."""
    codes, scales = pool
    bs = codes.shape[1]
    values = codes.view(torch.uint8)[ids].view(FP8).float()
    e = scales[ids][..., :bs].transpose(-1, -2).int() - 15
    return values.mul_(_power(e)[..., None])


def _attention(q, s, visible):
    """q [sequences, rows, heads, D] over the sequences' pages; visible [sequences, rows, keys]."""
    n, rows, hq, d = q.shape
    hkv = s["case"]["kv_heads"]
    ids = s["table"].long().clamp(min=0)
    q = q.float().view(n, rows, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(n, hkv, -1, d)
    k = _read(s["k"], ids).view(n, -1, hkv, d)
    scores = torch.matmul(q, k.permute(0, 2, 3, 1)).mul_(1.0 / math.sqrt(d))
    del k
    scores = scores.view(n, hkv, hq // hkv, rows, -1)
    scores.masked_fill_(~visible[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(top > -math.inf, top, 0.0)).exp_()
    total = scores.sum(-1, keepdim=True)
    v = _read(s["v"], ids).view(n, -1, hkv, d)
    out = torch.matmul(scores.view(n, hkv, (hq // hkv) * rows, -1), v.transpose(1, 2)).view(n, hkv, hq // hkv, rows, d)
    out = torch.where(total > 0, out / total, 0.0)
    return out.permute(0, 3, 1, 2, 4).reshape(n, rows, hq, d)


def _plain(s):
    case = s["case"]
    kind, dtype, bs = case["kind"], DTYPES[case["dtype"]], case["block_size"]
    if kind == "step":
        last = s["lens"].long() - 1
        slots = s["table"].long().gather(1, (last // bs)[:, None])[:, 0] * bs + last % bs
    else:
        slots = s["slots"]
    _store(s["k"], slots, s["k_new"])
    _store(s["v"], slots, s["v_new"])
    if kind == "cache":
        return [_read(s["k"], s["gather"].long()).to(dtype), _read(s["v"], s["gather"].long()).to(dtype), *s["k"], *s["v"]]
    pos = torch.arange(s["table"].shape[1] * bs, device="cuda")
    visible = (pos < s["lens"][:, None]) & (s["table"] >= 0).repeat_interleave(bs, 1)
    if kind == "step":
        out = _attention(s["q"].transpose(1, 2), s, visible[:, None]).to(dtype).transpose(1, 2)
        return [out, *s["k"], *s["v"]]
    cu, lens = (torch.from_numpy(x).long().cuda() for x in (s["cu"], s["host_lens"]))
    new = cu[1:] - cu[:-1]
    row = torch.arange(case["max_new"], device="cuda")
    visible = visible[:, None] & (row[:, None] < new[:, None, None])
    if case["causal"]:
        visible &= pos <= (lens - new)[:, None, None] + row[:, None]
    at = (cu[:-1, None] + row).clamp(max=s["q"].shape[0] - 1)
    out = _attention(s["q"][at], s, visible).to(dtype)
    return [out[row < new[:, None]], *s["k"], *s["v"]]


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def run(s):
    """The attention's output or the blocks read back, then the pools' codes and scales."""
    if not own:
        return _plain(s)
    from scicompute_attention_b200 import ops
    case = s["case"]
    if case["kind"] == "step":
        ops.kv_append_batched_fp8(s["k"], s["v"], s["k_new"], s["v_new"], s["table"], s["lens"])
        out = ops.paged_attention_fp8(s["q"], s["k"], s["v"], s["table"], s["lens"], block_size=case["block_size"], typical_len=s["mean"],
                                      longest_len=s["longest"])
        return [out, *s["k"], *s["v"]]
    ops.kv_append_fp8(s["k"], s["v"], s["k_new"], s["v_new"], s["slots"])
    if case["kind"] == "cache":
        dtype = DTYPES[case["dtype"]]
        return [ops.kv_gather_fp8(s["k"], s["gather"], dtype), ops.kv_gather_fp8(s["v"], s["gather"], dtype), *s["k"], *s["v"]]
    out = ops.flash_attention_paged_fp8(s["q"], s["k"], s["v"], s["table"], s["cu"], s["host_lens"], causal=case["causal"])
    return [out, *s["k"], *s["v"]]


# ------------------------------------------------------------------------------------------------
# 64 bits
# ------------------------------------------------------------------------------------------------
def _e4m3_numbers():
    """What the bytes 0 to 255 stand for: sign, 4 bits of exponent (bias 7), 3 of fraction; 127 and 255 are NaN."""
    def one(byte):
        size, fraction = byte >> 3 & 15, (byte & 7) / 8
        if size == 15 and byte & 7 == 7:
            return math.nan
        value = fraction * 2.0 ** -6 if size == 0 else (1 + fraction) * 2.0 ** (size - 7)
        return -value if byte & 128 else value
    return torch.tensor([one(b) for b in range(256)], dtype=torch.float64, device="cuda")


def _exact_pool(pool, slots, rows, numbers):
    """(bytes, exponents) of the pool after the rows have gone to the slots."""
    codes, scales = pool[0].view(torch.uint8).clone(), pool[1].clone()
    bs, hkv = codes.shape[1], codes.shape[2]
    x = rows.double()
    size = x.abs()
    most = torch.where(size.isnan(), 0.0, size).max(-1).values.clamp(max=57344.0)
    e = torch.full(most.shape, -14, dtype=torch.int64, device="cuda")
    for step in range(-14, 7):
        e += most > 448.0 * 2.0 ** step
    powers = torch.tensor([2.0 ** i for i in range(-14, 8)], dtype=torch.float64, device="cuda")
    size = (size / powers[e + 14][..., None]).clamp(max=448.0)
    positive = numbers[:127]
    middle = (positive[1:] + positive[:-1]) / 2
    at = torch.searchsorted(middle, size.contiguous())  # a tie goes to the lower one ...
    at += (at < 126) & (size == middle[at.clamp(max=125)]) & (at % 2 == 1)  # ... unless that is odd
    at = torch.where(x.isnan(), 127, at + 128 * torch.signbit(x))
    for h in range(hkv):
        codes[slots // bs, slots % bs, h] = at[:, h].to(torch.uint8)
        scales[slots // bs, h, slots % bs] = (e[:, h] + 15).to(torch.uint8)
    return codes, scales


def exact(case, seed):
    s = prepare(case, seed)
    bs, hkv, d = case["block_size"], case["kv_heads"], case["head_dim"]
    numbers = _e4m3_numbers()
    lens = s["lens"].tolist()
    if case["kind"] == "step":
        slots = torch.stack([s["table"][i, (n - 1) // bs].long() * bs + (n - 1) % bs for i, n in enumerate(lens)])
    else:
        slots = s["slots"].long()
    pools = [_exact_pool(s[x], slots, s[x + "_new"], numbers) for x in ("k", "v")]

    powers = torch.tensor([2.0 ** (i - 15) for i in range(23)], dtype=torch.float64, device="cuda")  # by the scale's byte

    def values(pool, blocks):
        codes, scales = pool
        return numbers[codes[blocks].long()] * powers[scales[blocks][:, :, :bs].permute(0, 2, 1).long()][..., None]

    stored = [x for codes, scales in pools for x in (codes.view(FP8), scales)]
    if case["kind"] == "cache":
        if case["gather"] * bs * hkv * d > 1 << 30:
            return [None, None, *stored]
        return [values(pools[0], s["gather"].long()), values(pools[1], s["gather"].long()), *stored]
    if work(case)["flops"] > 1e12:
        return [None, *stored]
    news = [1] * len(lens) if case["kind"] == "step" else np.diff(s["cu"]).tolist()
    flat = s["q"].reshape(-1, case["heads"], d)
    outs, first = [], 0
    for i, (n, new) in enumerate(zip(lens, news)):
        blocks = s["table"][i, :-(-n // bs)].long()
        k, v = (values(p, blocks).reshape(-1, hkv, d)[:n] for p in pools)
        q = flat[first:first + new].double()
        first += new
        out = torch.empty_like(q)
        group = case["heads"] // hkv
        for h in range(case["heads"]):
            scores = q[:, h] @ k[:, h // group].T / math.sqrt(d)
            if case.get("causal", True):
                hidden = torch.arange(n, device="cuda")[None, :] > torch.arange(n - new, n, device="cuda")[:, None]
                scores = scores.masked_fill(hidden, -math.inf)
            out[:, h] = torch.softmax(scores, -1) @ v[:, h // group]
        outs.append(out)
    return [torch.cat(outs).view(s["q"].shape), *stored]
