"""The operators of the 8-bit cache together, captured, on other streams, from several threads, inside guard zones, in pools beyond 32 bits."""
import ctypes as C
import threading

import numpy as np
import pytest
import torch

import fp8_reference as R
from test_fp8_decode_gpu import TYPES, make_pool, make_table, to_device
from test_guard_zones_gpu import Guarded

pytestmark = pytest.mark.gpu
HQ, HKV, D, BS = 8, 2, 128, 16


def _rand(*shape, dtype=torch.bfloat16, seed=0):
    return torch.randn(shape, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)).to(dtype)


def _near(out, q, cache, lens, new, kind):
    """`out` [T, H, D] against attention in 64 bits over the values `cache` = (k, v) [sequence][tokens, heads, D]."""
    at, got, q64 = 0, out.double().cpu().numpy(), q.double().cpu().numpy()
    for i, (n, m) in enumerate(zip(lens, new)):
        visible = np.arange(n)[None] <= n - m + np.arange(m)[:, None]
        for h in range(q64.shape[1]):
            want, bound = R.attention(q64[at:at + m, h], cache[0][i][:n, h // (HQ // HKV)], cache[1][i][:n, h // (HQ // HKV)], visible, 1 / np.sqrt(D), kind)
            assert (np.abs(got[at:at + m, h] - want) <= bound).all(), (i, h)
        at += m


@pytest.mark.parametrize("kind", TYPES)
def test_prompts_in_chunks_and_then_token_by_token(kind):
    """What a serving loop does: prompts enter in two chunks, each attended over as it comes, then tokens are decoded."""
    from scicompute_attention_b200 import ops
    dtype, prompts, width = TYPES[kind], [70, 333, 5], 24
    nblk = 3 * width
    k, v = ops.fp8_pool(nblk, BS, HKV, D), ops.fp8_pool(nblk, BS, HKV, D)
    table = torch.randperm(nblk, device="cuda").to(torch.int32).view(3, width).contiguous()
    kept = ([np.zeros((0, HKV, D))] * 3, [np.zeros((0, HKV, D))] * 3)
    lens, seed = [0, 0, 0], 1

    def stored(rows):
        codes, s = R.quantise(rows.double().cpu().numpy())
        return R.NUMBERS[codes] * 2.0 ** (s.astype(np.float64) - 15)[..., None]

    for part in (0, 1):
        new = [n // 2 if part == 0 else n - n // 2 for n in prompts]
        q, kn, vn = (_rand(sum(new), h, D, dtype=dtype, seed=seed + i) for i, h in enumerate((HQ, HKV, HKV)))
        seed += 3
        slots, at = [], 0
        for i, m in enumerate(new):
            pos = torch.arange(lens[i], lens[i] + m, device="cuda")
            slots.append(table[i, pos // BS] * BS + (pos % BS).to(torch.int32))
            for x, rows in zip(kept, (kn, vn)):
                x[i] = np.concatenate([x[i], stored(rows[at:at + m])])
            lens[i] += m
            at += m
        ops.kv_append_fp8(k, v, kn, vn, torch.cat(slots).to(torch.int32))
        cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        _near(ops.flash_attention_paged_fp8(q, k, v, table, cu, np.array(lens, np.int32)), q, kept, lens, new, kind)
    for _ in range(20):
        q, kn, vn = _rand(3, HQ, 1, D, dtype=dtype, seed=seed), _rand(3, HKV, D, dtype=dtype, seed=seed + 1), _rand(3, HKV, D, dtype=dtype, seed=seed + 2)
        seed += 3
        lens = [n + 1 for n in lens]
        for i in range(3):
            for x, rows in zip(kept, (kn, vn)):
                x[i] = np.concatenate([x[i], stored(rows[i:i + 1])])
        on_device = torch.tensor(lens, dtype=torch.int32, device="cuda")
        ops.kv_append_batched_fp8(k, v, kn, vn, table, on_device)
        out = ops.paged_attention_fp8(q, k, v, table, on_device, block_size=BS, typical_len=sum(lens) // 3, longest_len=max(lens))
        _near(out.view(3, HQ, D), q.view(3, HQ, D), kept, lens, [1] * 3, kind)
    for i, n in enumerate(lens):  # and everything can be read back
        back = ops.kv_gather_fp8(k, table[i].contiguous(), torch.float32).view(-1, HKV, D)[:n]
        assert np.array_equal(back.double().cpu().numpy(), kept[0][i])


def _work(seed, seqs=5, longest=900, d=D):
    """Everything a step and a chunk take, and the calls."""
    from scicompute_attention_b200 import ops
    rng = np.random.default_rng(seed)
    lens = [longest - 100 * i for i in range(seqs)]
    nblk = sum(-(-n // BS) for n in lens) + 2
    k, v = to_device(make_pool(rng, nblk, BS, HKV, d)), to_device(make_pool(rng, nblk, BS, HKV, d))
    table = torch.from_numpy(make_table(rng, lens, BS, nblk, -(-longest // BS) + 1)).cuda()
    dev_lens, host_lens = torch.tensor(lens, dtype=torch.int32, device="cuda"), np.array(lens, np.int32)
    cu = np.array([0, 1, 9, 40, 41, 130], np.int32)[:seqs + 1]
    q1, q, kn = _rand(seqs, HQ, 1, d, seed=seed), _rand(int(cu[-1]), HQ, d, seed=seed + 1), _rand(seqs, HKV, d, seed=seed + 2)
    slots = torch.randperm(nblk * BS, device="cuda")[:seqs].to(torch.int32)

    def call(stream=None):
        w = {} if stream is None else {"stream": stream}
        ops.kv_append_batched_fp8(k, v, kn, -kn, table, dev_lens, **w)
        ops.kv_append_fp8(k, v, kn, kn, slots, **w)
        return (ops.paged_attention_fp8(q1, k, v, table, dev_lens, block_size=BS, **w),
                ops.paged_attention_fp8(q1, k, v, table, dev_lens, block_size=BS, typical_len=800, longest_len=900, **w),
                ops.flash_attention_paged_fp8(q, k, v, table, cu, host_lens, **w), ops.kv_gather_fp8(k, table[0].contiguous(), torch.bfloat16, **w),
                ops.kv_gather_fp8(v, table[1].contiguous(), torch.float32, **w))
    return call, (q1, q, kn)


def _same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_the_native_forms_and_the_general_ones_give_the_same_bits():
    call, _ = _work(1)
    call()
    native = call()
    assert _same(native, call(torch.cuda.current_stream()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    on_side = call(side)
    side.synchronize()
    assert _same(native, on_side)


def test_a_captured_step_is_replayed_with_new_inputs():
    call, inputs = _work(2)
    call()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call()
    torch.cuda.synchronize()
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    call2, _ = _work(3, longest=700)
    expect2 = call2()
    with torch.cuda.graph(graph):
        got = call()
    with torch.cuda.graph(other):
        got2 = call2()
    for x in inputs:
        x.copy_(_rand(*x.shape, seed=77))
    graph.replay()
    other.replay()
    graph.replay()
    torch.cuda.synchronize()
    kept = [x.clone() for x in got]
    assert _same(call(), kept) and _same(got2, expect2)


def test_two_streams_and_threads_at_once():
    from scicompute_attention_b200 import ops
    works = [_work(10 + i, longest=700 + 50 * i)[0] for i in range(3)]
    expect = [w() for w in works]
    expect = [w() for w in works]
    torch.cuda.synchronize()
    got = [[] for _ in works]

    def run(work, into):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                into.append(work())
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=run, args=a) for a in zip(works, got)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for want, outs in zip(expect, got):
        assert len(outs) == 20 and all(_same(want, o) for o in outs)
    assert ops.flash_status() == 0


@pytest.mark.parametrize("d", [32, 96, 128, 256])
def test_writes_stay_inside_their_buffers(d):
    from scicompute_attention_b200 import _lib, ops
    lib, rng = _lib.lib(), np.random.default_rng(d)
    nblk, n = 5, 37
    pools = [(Guarded((nblk, BS, HKV, d), torch.uint8), Guarded((nblk, HKV, BS), torch.uint8)) for _ in range(2)]
    for codes, scales in pools:
        codes.tensor.zero_()
        scales.tensor.fill_(15)
    x = _rand(n, HKV, d, seed=d)
    slots = torch.from_numpy(rng.permutation(nblk * BS)[:n].astype(np.int32)).cuda()
    slots[:2] = torch.tensor([0, nblk * BS - 1], dtype=torch.int32)  # the first and the last
    slots[2:] = torch.from_numpy(rng.permutation(np.arange(1, nblk * BS - 1))[:n - 2].astype(np.int32)).cuda()
    (kc, ks), (vc, vs) = pools
    ops.kv_append_fp8((kc.tensor, ks.tensor), (vc.tensor, vs.tensor), x, x, slots)
    for g in (kc, ks, vc, vs):
        assert g.intact()
    shape = _lib.KvCacheShape(nblk, BS, HKV, d)
    ids = torch.tensor([4, 0, 7], dtype=torch.int32, device="cuda")
    for kind, dtype in ((0, torch.float32), (1, torch.float16), (2, torch.bfloat16)):
        out = Guarded((3, BS, HKV, d), dtype)
        _lib.check(lib.sca_launch_kv_gather_fp8(kc.tensor.data_ptr(), ks.tensor.data_ptr(), ids.data_ptr(), 3, out.tensor.data_ptr(), C.byref(shape), kind, None))
        torch.cuda.synchronize()
        assert out.intact() and torch.equal(out.tensor, ops.kv_gather_fp8((kc.tensor, ks.tensor), ids, dtype))
    table = torch.tensor([[0, 1, 2, -1], [3, 4, -1, -1]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([41, 32], dtype=torch.int32, device="cuda")
    q = _rand(2, HQ, 1, d, seed=d + 1)
    expect = ops.paged_attention_fp8(q, (kc.tensor, ks.tensor), (vc.tensor, vs.tensor), table, lens, block_size=BS)
    for splits in (1, 3):
        out, part = Guarded((2, HQ, 1, d), torch.bfloat16), Guarded((2 * HQ * splits * (2 + d),), torch.float32)
        p = _lib.DecodeFwdParams()
        base = 2 * HQ * splits
        p.q, p.k, p.v, p.out, p.page_table, p.seq_lens = q.data_ptr(), kc.tensor.data_ptr(), vc.tensor.data_ptr(), out.tensor.data_ptr(), table.data_ptr(), lens.data_ptr()
        at = part.tensor.data_ptr()
        p.partial_m, p.partial_l, p.partial_o = at, at + 4 * base, at + 8 * base
        p.batch, p.num_heads, p.num_kv_heads, p.seq_kv, p.head_dim, p.num_splits = 2, HQ, HKV, nblk * BS if splits > 1 else 100000, d, splits
        p.q_stride = p.o_stride = _lib.DecodeStrides(HQ * d, d, d)
        p.scale, p.dtype, p.block_size, p.max_blocks_per_seq, p.num_kv_blocks = ops.effective_scale(None, d), 2, BS, 4, nblk
        _lib.check(lib.sca_launch_paged_attention_fp8(C.byref(p), ks.tensor.data_ptr(), vs.tensor.data_ptr(), None, None))
        torch.cuda.synchronize()
        assert out.intact() and part.intact()
        assert (out.tensor.float() - expect.float()).abs().max() <= 2.0 ** -7 * expect.float().abs().max()  # two roundings of one number
    cu, host = np.array([0, 7, 39], np.int32), np.array([41, 32], np.int32)
    qc = _rand(39, HQ, d, seed=d + 2)
    out, ws = Guarded((39, HQ, d), torch.bfloat16), Guarded((int(lib.sca_flash_varlen_workspace_bytes(2, 39)),), torch.uint8)
    p = _lib.FlashPagedParams()
    p.q, p.out, p.k_pool, p.v_pool, p.page_table = qc.data_ptr(), out.tensor.data_ptr(), kc.tensor.data_ptr(), vc.tensor.data_ptr(), table.data_ptr()
    p.total_q, p.num_heads, p.num_kv_heads, p.head_dim, p.num_seqs, p.num_blocks, p.block_size, p.max_blocks_per_seq = 39, HQ, HKV, d, 2, nblk, BS, 4
    p.cu_seqlens_q, p.seq_lens_kv, p.scale, p.causal, p.dtype_id = cu.ctypes.data, host.ctypes.data, ops.effective_scale(None, d), 1, 2
    p.workspace, p.workspace_bytes = ws.tensor.data_ptr(), ws.tensor.numel()
    _lib.check(lib.sca_launch_flash_paged_fp8(C.byref(p), ks.tensor.data_ptr(), vs.tensor.data_ptr(), None))
    torch.cuda.synchronize()
    assert out.intact() and ws.intact()
    assert torch.equal(out.tensor, ops.flash_attention_paged_fp8(qc, (kc.tensor, ks.tensor), (vc.tensor, vs.tensor), table, cu, host))


def test_pools_beyond_32_bits():
    """Pools of more than 4 GiB: the pages of a sequence lie at both ends."""
    from scicompute_attention_b200 import ops
    hkv, d, bs = 8, 256, 64
    nblk = (1 << 32) // (bs * hkv * d) + 40
    k, v = ops.fp8_pool(nblk, bs, hkv, d), ops.fp8_pool(nblk, bs, hkv, d)
    small_k, small_v = ops.fp8_pool(4, bs, hkv, d), ops.fp8_pool(4, bs, hkv, d)
    far = torch.tensor([nblk - 1, 0, nblk - 33, 5], dtype=torch.int32, device="cuda")
    x, y = _rand(4 * bs, hkv, d, seed=1), _rand(4 * bs, hkv, d, seed=2)
    near_slots = torch.arange(4 * bs, dtype=torch.int32, device="cuda")
    ops.kv_append_fp8(small_k, small_v, x, y, near_slots)
    ops.kv_append_fp8(k, v, x, y, far[near_slots.long() // bs] * bs + near_slots % bs)
    near = torch.arange(4, dtype=torch.int32, device="cuda")
    for a, b in ((k, small_k), (v, small_v)):
        assert torch.equal(ops.kv_gather_fp8(a, far, torch.bfloat16), ops.kv_gather_fp8(b, near, torch.bfloat16))
    q1, q, lens = _rand(1, 16, 1, d, seed=3), _rand(70, 16, d, seed=4), torch.tensor([250], dtype=torch.int32, device="cuda")
    assert torch.equal(ops.paged_attention_fp8(q1, k, v, far[None], lens, block_size=bs, longest_len=250),
                       ops.paged_attention_fp8(q1, small_k, small_v, near[None], lens, block_size=bs, longest_len=250))
    cu, host = np.array([0, 70], np.int32), np.array([250], np.int32)
    assert torch.equal(ops.flash_attention_paged_fp8(q, k, v, far[None], cu, host), ops.flash_attention_paged_fp8(q, small_k, small_v, near[None], cu, host))
    ops.kv_append_batched_fp8(k, v, x[:1], y[:1], far[None], lens)
    ops.kv_append_batched_fp8(small_k, small_v, x[:1], y[:1], near[None], lens)
    assert torch.equal(ops.kv_gather_fp8(k, far, torch.float32), ops.kv_gather_fp8(small_k, near, torch.float32))
