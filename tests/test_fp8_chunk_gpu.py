"""Chunks of new tokens over the 8-bit paged cache against attention in 64 bits over the values the codes stand for."""
import numpy as np
import pytest
import torch

import fp8_reference as R
from test_fp8_decode_gpu import TYPES, keys_of, make_pool, make_table, to_device

pytestmark = pytest.mark.gpu


def run(q, k, v, table, cu, lens, **how):
    from scicompute_attention_b200 import ops
    out = ops.flash_attention_paged_fp8(q, to_device(k), to_device(v), torch.from_numpy(table).cuda(), cu, lens, **how)
    torch.cuda.synchronize()
    assert ops.flash_status() == 0
    return out


def check(out, q, k, v, table, cu, lens, bs, causal, scale, kind, rows=None):
    """`rows`: at most that many rows of a sequence, spread over it."""
    kv, vv = R.values(*k), R.values(*v)
    q64, got = q.double().cpu().numpy(), out.double().cpu().numpy()
    group = q64.shape[1] // kv.shape[2]
    for i, n in enumerate(lens):
        keys, there = keys_of(kv, table[i], n, bs)
        vals, _ = keys_of(vv, table[i], n, bs)
        new = cu[i + 1] - cu[i]
        at = np.arange(new) if rows is None or new <= rows else np.unique(np.linspace(0, new - 1, rows).astype(int))
        visible = there[None] & ((np.arange(n)[None] <= n - new + at[:, None]) if causal else True)
        for h in range(q64.shape[1]):
            want, bound = R.attention(q64[cu[i] + at, h], keys[:, h // group], vals[:, h // group], visible, scale, kind)
            off = np.abs(got[cu[i] + at, h] - want)
            assert (off <= bound).all(), (i, n, new, h, off.max(), np.argwhere(~(off <= bound))[:3])


def case(rng, lens, new, bs, hq, hkv, d, kind, spread=3):
    nblk = sum(-(-n // bs) for n in lens) + 3
    k, v = make_pool(rng, nblk, bs, hkv, d, spread), make_pool(rng, nblk, bs, hkv, d, spread)
    table = make_table(rng, lens, bs, nblk, -(-max(lens) // bs) + 1)
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    q = torch.from_numpy(rng.standard_normal((sum(new), hq, d))).to(TYPES[kind]).cuda()
    return q, k, v, table, cu, np.array(lens, np.int32)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("bs,hq,hkv,d", [(16, 8, 2, 128), (8, 4, 4, 128), (64, 8, 2, 64), (8, 6, 3, 32), (32, 4, 1, 256), (8, 2, 2, 256), (16, 4, 4, 96),
                                         (16, 2, 1, 192), (64, 3, 1, 160), (64, 16, 2, 256)])
def test_ragged_chunks(kind, causal, bs, hq, hkv, d):
    from scicompute_attention_b200 import ops
    rng = np.random.default_rng(bs + hq * 10 + d)
    lens, new = [1, 300, 129, 128, 257, 640, 17], [1, 3, 129, 1, 200, 70, 16]
    q, k, v, table, cu, lens = case(rng, lens, new, bs, hq, hkv, d, kind)
    out = run(q, k, v, table, cu, lens, causal=causal)
    assert out.shape == q.shape and out.dtype == q.dtype
    check(out, q, k, v, table, cu, lens, bs, causal, ops.effective_scale(None, d), kind)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("d,hq,hkv", [(128, 32, 8), (64, 32, 8), (256, 16, 4)])
def test_many_items_to_a_cta(kind, d, hq, hkv):
    """More query tiles than SMs: two tiles to an item, several items to a CTA, rings that go round many times."""
    from scicompute_attention_b200 import ops
    rng = np.random.default_rng(d)
    lens, new = [1500, 900, 40, 1300, 700], [1200, 900, 13, 37, 600]
    q, k, v, table, cu, lens = case(rng, lens, new, 16, hq, hkv, d, kind)
    out = run(q, k, v, table, cu, lens)
    check(out, q, k, v, table, cu, lens, 16, True, ops.effective_scale(None, d), kind, rows=40)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_one_item_shared_by_a_cluster(kind, d):
    """Few tokens against many keys: the CTAs of a cluster share the KV tiles."""
    from scicompute_attention_b200 import ops
    rng = np.random.default_rng(d + 1)
    q, k, v, table, cu, lens = case(rng, [3001, 1029], [37, 1], 16, 8, 2, d, kind)
    check(run(q, k, v, table, cu, lens), q, k, v, table, cu, lens, 16, True, ops.effective_scale(None, d), kind)


@pytest.mark.parametrize("d,bs", [(128, 8), (64, 16), (256, 64)])
def test_what_is_behind_a_sequence_or_in_holes_does_not_count(d, bs):
    """Holes - unmapped pages, pages outside the pool - weigh nothing; NaN codes and any scale byte behind the last token do no harm."""
    from scicompute_attention_b200 import ops
    rng = np.random.default_rng(d + 2)
    hq, hkv = 4, 2
    q, k, v, table, cu, lens = case(rng, [413, 77, 1000], [50, 77, 130], bs, hq, hkv, d, "bf16")
    nblk = k[0].shape[0]
    live = np.zeros((nblk, bs), bool)
    for i, n in enumerate(lens):
        live[table[i, np.arange(n) // bs], np.arange(n) % bs] = True
    for codes, scales in (k, v):
        codes[~live] = 127
        scales[:, :, :bs][~np.repeat(live[:, None], hkv, 1)] = 255
        scales[:, :, bs:] = 255
    table[0, 2], table[2, 1], table[2, 5], table[2, 6] = -1, nblk, nblk + 100, -7
    out = run(q, k, v, table, cu, lens, causal=False)
    check(out, q, k, v, table, cu, lens, bs, False, ops.effective_scale(None, d), "bf16")


def test_a_row_that_sees_nothing_is_zero():
    rng = np.random.default_rng(3)
    q, k, v, table, cu, lens = case(rng, [100, 40], [9, 40], 16, 4, 2, 128, "fp16")
    table[0] = -1
    out = run(q, k, v, table, cu, lens)
    assert not out[:9].any() and out[9:].any()
    table[1, 0] = -1  # the first 16 rows of the second sequence lose all of their keys
    out = run(q, k, v, table, cu, lens)
    assert not out[9:25].any() and out[25:].any(-1).all()


@pytest.mark.parametrize("d,size", [(128, 1e-30), (64, 1e-4), (256, 300.0), (128, 1e30)])
def test_bf16_queries_of_any_size(d, size):
    from scicompute_attention_b200 import ops
    rng = np.random.default_rng(17)
    q, k, v, table, cu, lens = case(rng, [300, 200], [60, 150], 16, 4, 2, d, "bf16", spread=0)
    q = (q.double() * size).to(torch.bfloat16)
    q[5] = 0
    q[20:30] = (q[20:30].double() * 1e-3).to(torch.bfloat16)
    scale = float(np.float32(0.1 / size))
    check(run(q, k, v, table, cu, lens, scale=scale), q, k, v, table, cu, lens, 16, True, scale, "bf16")


def test_values_of_very_different_sizes():
    from scicompute_attention_b200 import ops
    rng = np.random.default_rng(18)
    q, k, v, table, cu, lens = case(rng, [500], [140], 16, 2, 1, 128, "fp16", spread=0)
    v = make_pool(rng, k[0].shape[0], 16, 1, 128, spread=12)
    check(run(q, k, v, table, cu, lens), q, k, v, table, cu, lens, 16, True, ops.effective_scale(None, 128), "fp16")


def test_the_same_call_gives_the_same_bits():
    rng = np.random.default_rng(19)
    q, k, v, table, cu, lens = case(rng, [2000, 1500, 300], [700, 1500, 20], 16, 32, 8, 128, "bf16")
    first = run(q, k, v, table, cu, lens)
    for _ in range(30):
        assert torch.equal(run(q, k, v, table, cu, lens), first)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("lens,new", [([3001], [37]), ([3001, 500] * 8, [300, 500] * 8)])
def test_a_query_of_nan_gives_nan(kind, lens, new):
    rng = np.random.default_rng(22)
    q, k, v, table, cu, lens = case(rng, lens, new, 16, 8, 2, 128, kind)
    want = run(q, k, v, table, cu, lens)
    q[20, 3] = float("nan")
    got = run(q, k, v, table, cu, lens)
    assert got[20, 3].isnan().all()
    got[20, 3] = want[20, 3]
    assert torch.equal(got, want)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("seqs", [3, 85, 86, 200])
def test_work_lists_of_any_length(seqs, d):
    """Lists of up to 2 KB (85 sequences of one entry) go with the launch, longer ones - and those of whole D=64 items - ahead of it."""
    from scicompute_attention_b200 import ops
    rng = np.random.default_rng(23)
    new = [1 + i % 7 for i in range(seqs)]
    q, k, v, table, cu, lens = case(rng, [n + 11 * (i % 5) for i, n in enumerate(new)], new, 16, 4, 2, d, "fp16")
    check(run(q, k, v, table, cu, lens), q, k, v, table, cu, lens, 16, True, ops.effective_scale(None, d), "fp16")
