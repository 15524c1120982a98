"""The two-kernel form of the 8-bit decode - parts of a sequence, then their merge - for every head dim, both kinds of merge and more than eight heads to
a kv head, against attention in 64 bits over the values the codes stand for."""
import ctypes as C

import numpy as np
import pytest
import torch

import fp8_reference as R
from test_fp8_decode_gpu import TYPES, check, keys_of, make_pool, make_table, to_device

pytestmark = pytest.mark.gpu
GROUPS = [(4, 2), (6, 1), (32, 2), (24, 1), (40, 1)]


def decode(q, k, v, table, lens, block_size, splits, scale):
    """The C entry with `splits` slots to a row, NaN in the scratch, sized for a call that is not one for clusters."""
    from scicompute_attention_b200 import _lib, ops
    seqs, hq, _, d = q.shape
    rows = seqs * hq * splits
    part, out = torch.full((-(-2 * rows // 4) * 4 + rows * d,), float("nan"), device="cuda"), torch.full_like(q, float("nan"))
    p = _lib.DecodeFwdParams()
    p.q, p.k, p.v, p.out, p.page_table, p.seq_lens = q.data_ptr(), k.codes.data_ptr(), v.codes.data_ptr(), out.data_ptr(), table.data_ptr(), lens.data_ptr()
    at = part.data_ptr()
    p.partial_m, p.partial_l, p.partial_o = at, at + 4 * rows, at + 4 * (-(-2 * rows // 4) * 4)
    p.batch, p.num_heads, p.num_kv_heads, p.seq_kv, p.head_dim, p.num_splits = seqs, hq, k.codes.shape[2], table.shape[1] * block_size, d, splits
    p.q_stride = p.o_stride = _lib.DecodeStrides(hq * d, d, d)
    p.scale, p.dtype, p.block_size, p.max_blocks_per_seq, p.num_kv_blocks = scale, ops.dtype_id(q.dtype), block_size, table.shape[1], k.codes.shape[0]
    cluster = C.c_int32(-1)
    _lib.check(_lib.lib().sca_launch_paged_attention_fp8(C.byref(p), k.scales.data_ptr(), v.scales.data_ptr(), C.byref(cluster), None))
    assert cluster.value == 0
    return out


def case(seed, lens, hq, hkv, d, bs, kind, width):
    rng = np.random.default_rng(seed)
    nblk = sum(-(-n // bs) for n in lens) + 3
    k, v = make_pool(rng, nblk, bs, hkv, d), make_pool(rng, nblk, bs, hkv, d)
    table = make_table(rng, lens, bs, nblk, width)
    return torch.from_numpy(rng.standard_normal((len(lens), hq, 1, d))).to(TYPES[kind]).cuda(), k, v, table


def expected(q, k, v, table, lens, bs, scale, kind):
    """Attention in 64 bits and how far a kernel may be from it, [sequences, heads, D] each; nothing where no token is there."""
    kv, vv, q64 = R.values(*k), R.values(*v), q[:, :, 0].double().cpu().numpy()
    want, bound = np.zeros_like(q64), np.zeros_like(q64)
    group = q64.shape[1] // kv.shape[2]
    for i, n in enumerate(lens):
        keys, there = keys_of(kv, table[i], n, bs)
        vals, _ = keys_of(vv, table[i], n, bs)
        for h in range(kv.shape[2] if there.any() else 0):
            rows = slice(h * group, (h + 1) * group)
            want[i, rows], bound[i, rows] = R.attention(q64[i, rows], keys[:, h], vals[:, h], np.repeat(there[None], group, 0), scale, kind)
    return want, bound


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("hq,hkv", GROUPS)
@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 192, 256])
def test_every_geometry(kind, hq, hkv, d):
    """Sequences in one part, in a few, in many; one without a token, one whose pages are holes, one with holes inside. Rows of one slot, of up to
    eight (a warp merges a row), of more (the eight warps of a CTA do)."""
    from scicompute_attention_b200 import ops
    bs, lens, scale = 16, [1700, 1, 0, 129, 700, 33, 64], ops.effective_scale(None, d)
    q, k, v, table = case(hq * 1000 + d, lens, hq, hkv, d, bs, kind, 7000)
    table[0, 5], table[0, 80:84], table[4, 2] = -1, -1, k[0].shape[0] + 9
    table[6] = -1
    on_device = to_device(k), to_device(v), torch.from_numpy(table).cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    want, bound = expected(q, k, v, table, lens, bs, scale, kind)
    for splits in (1, 5, 8, 9, 60):
        off = np.abs(decode(q, *on_device, bs, splits, scale)[:, :, 0].double().cpu().numpy() - want)
        assert (off <= bound).all(), (splits, off.max())


@pytest.mark.parametrize("hq,hkv", [(16, 2), (40, 1)])
@pytest.mark.parametrize("d", [32, 96, 160, 256])
def test_many_rows(hq, hkv, d):
    """More rows than the merge of eight warps to a row is for, and more sequences than CTAs."""
    from scicompute_attention_b200 import ops
    bs, lens = 8, [[60, 3, 130, 0][i % 4] + i % 5 for i in range(700)]
    q, k, v, table = case(d, lens, hq, hkv, d, bs, "bf16", -(-max(lens) // bs) + 2)
    scale, few = ops.effective_scale(None, d), [0, 1, 2, 3, 349, 695, 698, 699]
    out = decode(q, to_device(k), to_device(v), torch.from_numpy(table).cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), bs, 9, scale)
    check(out[few], q[few], k, v, table[few], [lens[i] for i in few], bs, scale, "bf16")
    hints = dict(typical_len=sum(lens) // len(lens), longest_len=max(lens))
    out, stats = ops.paged_attention_fp8(q, to_device(k), to_device(v), torch.from_numpy(table).cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), block_size=bs,
                                         return_stats=True, **hints)
    assert stats["cluster"] == 0
    check(out[few], q[few], k, v, table[few], [lens[i] for i in few], bs, scale, "bf16")


@pytest.mark.parametrize("hq,hkv,d,n", [(16, 1, 64, 140_000), (8, 1, 128, 100_003), (16, 1, 256, 60_001)])
def test_one_long_sequence(hq, hkv, d, n):
    """One sequence on every CTA of the machine: with and without hints, through the native and the general form."""
    from scicompute_attention_b200 import ops
    bs = 32
    q, k, v, table = case(n, [n], hq, hkv, d, bs, "fp16", -(-n // bs))
    args = q, to_device(k), to_device(v), torch.from_numpy(table).cuda(), torch.tensor([n], dtype=torch.int32).cuda()
    want, bound = expected(q, k, v, table, [n], bs, ops.effective_scale(None, d), "fp16")
    for hints in ({}, dict(typical_len=n, longest_len=n)):
        out, stats = ops.paged_attention_fp8(*args, block_size=bs, return_stats=True, **hints)
        assert stats["cluster"] == 0 and (np.abs(out[:, :, 0].double().cpu().numpy() - want) <= bound).all()
        assert torch.equal(ops.paged_attention_fp8(*args, block_size=bs, **hints), out)
