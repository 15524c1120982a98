"""Paged decode over the 8-bit cache against attention in 64 bits over the values the codes stand for."""
import numpy as np
import pytest
import torch

import fp8_reference as R

pytestmark = pytest.mark.gpu
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def make_pool(rng, nblk, bs, hkv, d, spread=3):
    """Codes of any size but NaN, scales of any size within 2^spread of each other; both as numpy arrays."""
    x = rng.standard_normal((nblk, bs, hkv, d)) * 2.0 ** rng.integers(-spread, spread + 1, (nblk, bs, hkv, 1))
    codes, s = R.quantise(x)
    scales = rng.integers(1, 23, (nblk, hkv, R.scale_row(bs)), dtype=np.uint8)
    scales[:, :, :bs] = s.transpose(0, 2, 1)
    return codes, scales


def to_device(pool):
    from scicompute_attention_b200 import ops
    return ops.Fp8Pool(torch.from_numpy(pool[0]).cuda().view(torch.float8_e4m3fn), torch.from_numpy(pool[1]).cuda())


def make_table(rng, lens, bs, nblk, width):
    """Pages of every sequence out of a shuffled pool, -1 behind the last."""
    ids, at = rng.permutation(nblk), 0
    table = np.full((len(lens), width), -1, np.int32)
    for i, n in enumerate(lens):
        pages = -(-n // bs)
        table[i, :pages] = ids[at:at + pages]
        at += pages
    return table


def keys_of(pool_values, table_row, n, bs):
    """(values [n, heads, D], which of the n tokens there are)."""
    page = table_row[np.arange(n) // bs]
    there = (page >= 0) & (page < pool_values.shape[0])
    return pool_values[np.where(there, page, 0), np.arange(n) % bs], there


def check(out, q, k, v, table, lens, bs, scale, kind):
    kv, vv = R.values(*k), R.values(*v)
    q64, got = q.double().cpu().numpy(), out.double().cpu().numpy()
    group = q64.shape[1] // kv.shape[2]
    for i, n in enumerate(lens):
        keys, there = keys_of(kv, table[i], n, bs)
        vals, _ = keys_of(vv, table[i], n, bs)
        for h in range(q64.shape[1]):
            if not there.any():
                assert not got[i, h].any()
                continue
            want, bound = R.attention(q64[i, h], keys[:, h // group], vals[:, h // group], there[None], scale, kind)
            assert (np.abs(got[i, h] - want) <= bound).all(), (i, n, h, np.abs(got[i, h] - want).max(), bound.min())


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("hq,hkv,d", [(8, 8, 128), (32, 8, 128), (16, 2, 64), (32, 2, 128), (24, 1, 96), (6, 3, 32), (10, 1, 160), (4, 2, 192),
                                      (16, 2, 256), (32, 2, 256), (40, 1, 64)])
@pytest.mark.parametrize("bs", [16, 4, 40])
def test_ragged_batch(kind, hq, hkv, d, bs):
    from scicompute_attention_b200 import ops
    rng = np.random.default_rng(hq * 100 + d + bs)
    lens = [1, 31, 32, 33, 128, 129, 513, 700, 0, 2]
    nblk = sum(-(-n // bs) for n in lens) + 3
    k, v = make_pool(rng, nblk, bs, hkv, d), make_pool(rng, nblk, bs, hkv, d)
    table = make_table(rng, lens, bs, nblk, -(-max(lens) // bs) + 1)
    table[6, 3], table[7, 5] = -1, nblk + 7  # holes: unmapped, outside the pool
    q = torch.from_numpy(rng.standard_normal((len(lens), hq, 1, d))).to(TYPES[kind]).cuda()
    out = ops.paged_attention_fp8(q, to_device(k), to_device(v), torch.from_numpy(table).cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), block_size=bs)
    assert out.shape == q.shape and out.dtype == q.dtype
    check(out, q, k, v, table, lens, bs, ops.effective_scale(None, d), kind)


@pytest.mark.parametrize("hints", [True, False])
@pytest.mark.parametrize("lens,clusters", [([5], True), ([1000], True), ([40000, 3], False), ([700] * 300, False), ([60] * 300, False), ([1, 127] * 200, False)])
def test_both_ways_of_launching(lens, clusters, hints):
    from scicompute_attention_b200 import ops
    rng = np.random.default_rng(len(lens))
    bs, hq, hkv, d = 16, 8, 2, 128
    nblk = sum(-(-n // bs) for n in lens)
    k, v = make_pool(rng, nblk, bs, hkv, d), make_pool(rng, nblk, bs, hkv, d)
    table = make_table(rng, lens, bs, nblk, -(-max(lens) // bs))
    q = torch.from_numpy(rng.standard_normal((len(lens), hq, 1, d))).to(torch.float16).cuda()
    out, stats = ops.paged_attention_fp8(q, to_device(k), to_device(v), torch.from_numpy(table).cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                                         block_size=bs, return_stats=True, **(dict(typical_len=sum(lens) // len(lens), longest_len=max(lens)) if hints else {}))
    assert (stats["cluster"] > 0) == clusters
    few = range(0, len(lens), max(1, len(lens) // 4))
    check(out[list(few)], q[list(few)], k, v, table[list(few)], [lens[i] for i in few], bs, ops.effective_scale(None, d), "fp16")


def test_what_lies_behind_a_sequence_does_not_count():
    """NaN codes and any scale byte behind a sequence's last token, in unmapped pages and in the scales' padding."""
    from scicompute_attention_b200 import ops
    rng = np.random.default_rng(5)
    bs, hq, hkv, d, lens = 8, 4, 2, 64, [13, 1, 50]
    nblk = 20
    k, v = make_pool(rng, nblk, bs, hkv, d), make_pool(rng, nblk, bs, hkv, d)
    table = make_table(rng, lens, bs, nblk, 9)
    for codes, scales in (k, v):
        live = np.zeros((nblk, bs), bool)
        for i, n in enumerate(lens):
            live[table[i, np.arange(n) // bs], np.arange(n) % bs] = True
        codes[~live] = 127
        scales[:, :, :bs][~np.repeat(live[:, None], hkv, 1)] = 255
        scales[:, :, bs:] = 255
    q = torch.from_numpy(rng.standard_normal((3, hq, 1, d))).to(torch.bfloat16).cuda()
    out = ops.paged_attention_fp8(q, to_device(k), to_device(v), torch.from_numpy(table).cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), block_size=bs)
    check(out, q, k, v, table, lens, bs, ops.effective_scale(None, d), "bf16")


@pytest.mark.parametrize("kind,size", [("bf16", 1e-30), ("bf16", 1e-4), ("bf16", 300.0), ("bf16", 1e30), ("fp16", 2e-5), ("fp16", 900.0)])
def test_queries_of_any_size(kind, size):
    """bf16 queries are carried as fp16 numbers times a power of two per head. The scale undoes their size."""
    from scicompute_attention_b200 import ops
    rng = np.random.default_rng(11)
    bs, hq, hkv, d, lens = 16, 8, 2, 128, [300, 77]
    k, v = make_pool(rng, 30, bs, hkv, d, spread=0), make_pool(rng, 30, bs, hkv, d)
    table = make_table(rng, lens, bs, 30, 20)
    q = torch.from_numpy(rng.standard_normal((2, hq, 1, d)) * size).to(TYPES[kind]).cuda()
    q[1, 3] = 0
    scale = float(np.float32(0.1 / size))
    out = ops.paged_attention_fp8(q, to_device(k), to_device(v), torch.from_numpy(table).cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), block_size=bs,
                                  scale=scale)
    check(out, q, k, v, table, lens, bs, scale, kind)


def test_values_of_very_different_sizes():
    """Rows of V from the smallest scale to the largest: each keeps its weight."""
    from scicompute_attention_b200 import ops
    rng = np.random.default_rng(12)
    bs, d, n = 16, 64, 200
    k, v = make_pool(rng, 13, bs, 1, d, spread=0), make_pool(rng, 13, bs, 1, d, spread=12)
    table = np.arange(13, dtype=np.int32)[None]
    q = torch.from_numpy(rng.standard_normal((1, 5, 1, d))).to(torch.float16).cuda()
    out = ops.paged_attention_fp8(q, to_device(k), to_device(v), torch.from_numpy(table).cuda(), torch.tensor([n], dtype=torch.int32).cuda(), block_size=bs)
    check(out, q, k, v, table, [n], bs, ops.effective_scale(None, d), "fp16")


def test_without_lengths_the_whole_table_is_read():
    from scicompute_attention_b200 import ops
    rng = np.random.default_rng(13)
    k, v = make_pool(rng, 12, 16, 2, 64), make_pool(rng, 12, 16, 2, 64)
    table = rng.permutation(12).reshape(2, 6).astype(np.int32)
    q = torch.from_numpy(rng.standard_normal((2, 4, 1, 64))).to(torch.bfloat16).cuda()
    out = ops.paged_attention_fp8(q, to_device(k), to_device(v), torch.from_numpy(table).cuda(), None, block_size=16)
    check(out, q, k, v, table, [96, 96], 16, ops.effective_scale(None, 64), "bf16")


@pytest.mark.parametrize("hints", [dict(typical_len=1), dict(typical_len=5000, longest_len=1), dict(longest_len=100000), dict(typical_len=3, longest_len=3)])
def test_wrong_hints_cost_time_only(hints):
    from scicompute_attention_b200 import ops
    rng = np.random.default_rng(14)
    lens = [3, 900, 40, 2000] * 30
    nblk = sum(-(-n // 16) for n in lens)
    k, v = make_pool(rng, nblk, 16, 2, 64), make_pool(rng, nblk, 16, 2, 64)
    table = make_table(rng, lens, 16, nblk, -(-max(lens) // 16))
    q = torch.from_numpy(rng.standard_normal((len(lens), 4, 1, 64))).to(torch.float16).cuda()
    out = ops.paged_attention_fp8(q, to_device(k), to_device(v), torch.from_numpy(table).cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), block_size=16, **hints)
    check(out[:8], q[:8], k, v, table[:8], lens[:8], 16, ops.effective_scale(None, 64), "fp16")
    check(out[-4:], q[-4:], k, v, table[-4:], lens[-4:], 16, ops.effective_scale(None, 64), "fp16")


def test_nan_of_a_token_that_counts_is_seen():
    from scicompute_attention_b200 import ops
    k, v = ops.fp8_pool(4, 16, 1, 64), ops.fp8_pool(4, 16, 1, 64)
    x = torch.randn(20, 1, 64, device="cuda", dtype=torch.float16)
    y = x.clone()
    y[7, 0, 5] = float("nan")
    ops.kv_append_fp8(k, v, x, y, torch.arange(20, dtype=torch.int32, device="cuda"))
    table, lens = torch.arange(4, dtype=torch.int32, device="cuda")[None], torch.tensor([20], dtype=torch.int32, device="cuda")
    out = ops.paged_attention_fp8(x[:1].view(1, 1, 1, 64), k, v, table, lens, block_size=16)
    assert out.isnan().view(-1).nonzero().view(-1).tolist() == [5]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("lens,cluster", [([300, 40], True), ([40000, 40], False)])
def test_a_query_of_nan_gives_nan(kind, lens, cluster):
    """Every score of the row is NaN, and so is what comes out, in parts or in one piece; the others keep their numbers."""
    from scicompute_attention_b200 import ops
    rng = np.random.default_rng(21)
    nblk = sum(-(-n // 16) for n in lens)
    k, v = to_device(make_pool(rng, nblk, 16, 2, 128)), to_device(make_pool(rng, nblk, 16, 2, 128))
    table = torch.from_numpy(make_table(rng, lens, 16, nblk, -(-max(lens) // 16))).cuda()
    q = torch.from_numpy(rng.standard_normal((2, 8, 1, 128))).to(TYPES[kind]).cuda()
    run = lambda: ops.paged_attention_fp8(q, k, v, table, torch.tensor(lens, dtype=torch.int32).cuda(), block_size=16, return_stats=True)
    want, stats = run()
    assert (stats["cluster"] > 0) == cluster
    q[0, 3] = float("nan")
    got, _ = run()
    assert got[0, 3].isnan().all()
    got[0, 3] = want[0, 3]
    assert torch.equal(got, want)
