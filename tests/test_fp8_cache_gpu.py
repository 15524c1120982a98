"""The 8-bit KV cache as it is written and read back: bit for bit what the definition in 64 bits says."""
import numpy as np
import pytest
import torch

import fp8_reference as R

pytestmark = pytest.mark.gpu
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _rows(rng, n, hkv, d, dtype):
    """Rows of very different sizes, with zeros, numbers next to the borders of the scales, ties and what cannot be stored."""
    x = rng.standard_normal((n, hkv, d)) * 2.0 ** rng.integers(-22, 15, (n, hkv, 1))
    x.reshape(-1)[::17] *= 2.0 ** -8
    x = torch.from_numpy(x).to(dtype)
    flat = x.view(-1, d)
    flat[0] = 0.0
    for i, most in enumerate((448.0, 449.0, 450.0, 0.02734375, 0.0275, 57344.0, 60000.0)):  # 448 * 2^e and just above it
        if i + 1 < flat.shape[0]:
            flat[i + 1] = (torch.arange(d) / d * most).to(dtype)
            flat[i + 1, d // 2] = -most
    if flat.shape[0] > 12:
        flat[8, :8] = torch.tensor([1.0625, 1.1875, -1.0625, 1.3125, 17.0, 19.0, 0.0009765625, -0.0])  # halfway between two codes
        flat[9, 3], flat[9, 5] = float("inf"), float("-inf")
        flat[10, 2] = float("nan")
        flat[11] = float("nan")
    return x


def _same(got, want):
    """Codes are equal, a NaN being a NaN under either sign."""
    return np.array_equal(got, want) or np.array_equal(R.NUMBERS[got], R.NUMBERS[want], equal_nan=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bs,hkv,d", [(1, 1, 16), (8, 2, 64), (16, 8, 128), (5, 3, 48), (64, 1, 256), (32, 2, 96), (16, 3, 176), (24, 5, 32)])
def test_written_and_read_back(dtype, bs, hkv, d):
    from scicompute_attention_b200 import ops
    rng = np.random.default_rng(bs * 1000 + d)
    nblk, n = 9, 3 * bs + 13 if bs < 64 else 150
    n = min(n, nblk * bs)
    k_new, v_new = _rows(rng, n, hkv, d, TYPES[dtype]), _rows(rng, n, hkv, d, TYPES[dtype])
    slots = rng.permutation(nblk * bs)[:n].astype(np.int32)
    slots[0] = -1
    if n > 3:
        slots[3] = nblk * bs
    pools, want = [], []
    for new in (k_new, v_new):
        codes, scales = rng.integers(0, 127, (nblk, bs, hkv, d), dtype=np.uint8), rng.integers(1, 23, (nblk, hkv, R.scale_row(bs)), dtype=np.uint8)
        pools.append(ops.Fp8Pool(torch.from_numpy(codes.copy()).cuda().view(torch.float8_e4m3fn), torch.from_numpy(scales.copy()).cuda()))
        c, s = R.quantise(new.double().numpy())
        for i, slot in enumerate(slots):
            if 0 <= slot < nblk * bs:
                codes[slot // bs, slot % bs], scales[slot // bs, :, slot % bs] = c[i], s[i]
        want.append((codes, scales))
    ops.kv_append_fp8(*pools, k_new.cuda(), v_new.cuda(), torch.from_numpy(slots).cuda())
    ids = np.array([3, 0, -1, nblk, 8, 3], np.int32)
    for pool, (codes, scales) in zip(pools, want):
        assert _same(pool.codes.view(torch.uint8).cpu().numpy(), codes)
        assert np.array_equal(pool.scales.cpu().numpy(), scales)
        stands_for = R.values(codes, scales)
        for out_type in TYPES.values():
            got = ops.kv_gather_fp8(pool, torch.from_numpy(ids).cuda(), out_type)
            assert got.shape == (ids.size, bs, hkv, d) and got.dtype == out_type
            for i, b in enumerate(ids):  # exact in every type
                assert np.array_equal(got[i].double().cpu().numpy(), stands_for[b] if 0 <= b < nblk else np.zeros((bs, hkv, d)), equal_nan=True)


def test_what_is_stored_is_near():
    """The distance of a stored number from the one that came: half a step of 4 bits, or half of the smallest step."""
    from scicompute_attention_b200 import ops
    x = (torch.randn(300, 4, 128, generator=torch.Generator().manual_seed(3)) * 3).to(torch.bfloat16)
    pool = ops.fp8_pool(19, 16, 4, 128)
    ops.kv_append_fp8(pool, ops.fp8_pool(19, 16, 4, 128), x.cuda(), x.cuda(), torch.arange(300, dtype=torch.int32, device="cuda"))
    back = ops.kv_gather_fp8(pool, torch.arange(19, dtype=torch.int32, device="cuda"), torch.float32).view(-1, 4, 128)
    smallest = 2.0 ** (pool.scales.view(19, 4, 16).transpose(1, 2).reshape(-1, 4, 1).float() - 15) * 2.0 ** -10
    assert ((back[:300].cpu() - x.float()).abs() <= torch.maximum(x.float().abs() * 2.0 ** -4, smallest[:300].cpu())).all()
    assert not back[300:].any()


@pytest.mark.parametrize("bs,width", [(16, 5), (8, 9), (3, 30)])
def test_one_token_per_sequence(bs, width):
    from scicompute_attention_b200 import ops
    rng = np.random.default_rng(bs)
    hkv, d = 2, 64
    lens = np.array([1, bs, bs + 1, 0, 2 * bs + 2, width * bs + 5, 3, -4], np.int32)  # none, past the table
    nblk = len(lens) * width + 2
    table = rng.permutation(nblk)[:len(lens) * width].reshape(len(lens), width).astype(np.int32)
    table[4, 2], table[6, 0] = -1, nblk  # unmapped, outside the pool
    x = _rows(rng, len(lens), hkv, d, torch.bfloat16)
    k, v = ops.fp8_pool(nblk, bs, hkv, d), ops.fp8_pool(nblk, bs, hkv, d)
    ops.kv_append_batched_fp8(k, v, x.cuda(), (-x).cuda(), torch.from_numpy(table).cuda(), torch.from_numpy(lens).cuda())
    codes, scales = np.zeros((nblk, bs, hkv, d), np.uint8), np.full((nblk, hkv, R.scale_row(bs)), 15, np.uint8)
    c, s = R.quantise(x.double().numpy())
    written = set()
    for i, n in enumerate(lens):
        if n < 1 or (n - 1) // bs >= width or not 0 <= table[i, (n - 1) // bs] < nblk:
            continue
        at = (table[i, (n - 1) // bs], (n - 1) % bs)
        assert at not in written
        written.add(at)
        codes[at], scales[at[0], :, at[1]] = c[i], s[i]
    assert _same(k.codes.view(torch.uint8).cpu().numpy(), codes) and np.array_equal(k.scales.cpu().numpy(), scales)
    assert np.array_equal(v.scales.cpu().numpy(), scales)
    assert np.array_equal(R.NUMBERS[v.codes.view(torch.uint8).cpu().numpy()], -R.NUMBERS[codes] + 0.0, equal_nan=True)


def test_rows_that_start_anywhere():
    """New K / V need not lie on 16-byte boundaries."""
    from scicompute_attention_b200 import ops
    x = torch.randn(40 * 2 * 64 + 3, device="cuda").to(torch.float16)
    slots = torch.randperm(48, device="cuda").to(torch.int32)[:40]
    a, b, other = (ops.fp8_pool(3, 16, 2, 64) for _ in range(3))
    ops.kv_append_fp8(a, other, x[3:].view(40, 2, 64), x[3:].view(40, 2, 64), slots)
    ops.kv_append_fp8(b, other, x[3:].clone().view(40, 2, 64), x[3:].clone().view(40, 2, 64), slots)
    assert torch.equal(a.codes.view(torch.uint8), b.codes.view(torch.uint8)) and torch.equal(a.scales, b.scales)
    assert torch.equal(a.codes.view(torch.uint8), other.codes.view(torch.uint8))


def test_freed_blocks_read_as_zeros():
    from scicompute_attention_b200 import ops
    k, v = ops.fp8_pool(4, 16, 2, 64), ops.fp8_pool(4, 16, 2, 64)
    x = torch.randn(64, 2, 64, device="cuda", dtype=torch.bfloat16)
    ops.kv_append_fp8(k, v, x, x, torch.arange(64, dtype=torch.int32, device="cuda"))
    ids = torch.tensor([1, 3], dtype=torch.int32, device="cuda")
    ops.kv_reset(k.codes, v.codes, ids)
    assert not ops.kv_gather_fp8(k, ids, torch.float16).any() and not ops.kv_gather_fp8(v, ids, torch.float16).any()
    assert ops.kv_gather_fp8(k, torch.tensor([0, 2], dtype=torch.int32, device="cuda"), torch.float16).any()


def test_nothing_to_do():
    from scicompute_attention_b200 import ops
    k, v = ops.fp8_pool(2, 16, 1, 32), ops.fp8_pool(2, 16, 1, 32)
    none = torch.empty(0, 1, 32, device="cuda", dtype=torch.float16)
    ints = torch.empty(0, dtype=torch.int32, device="cuda")
    ops.kv_append_fp8(k, v, none, none, ints)
    ops.kv_append_batched_fp8(k, v, none, none, torch.empty(0, 3, dtype=torch.int32, device="cuda"), ints)
    assert ops.kv_gather_fp8(k, ints, torch.float16).shape == (0, 16, 1, 32)
