"""Tensors on the host are refused by the operators of a paged cache that stays small - whole calls of them, and each tensor alone - where the same call is
served otherwise."""
import numpy as np
import pytest
import torch

from scicompute_attention_b200 import _lib, ops

B, HQ, HKV, D, BS, W = 2, 4, 2, 64, 16, 4
CU, NEW, TOTAL, PREFIX = (np.array(x, np.int32) for x in ([0, 2], [0, 4, 9], [20, 20], [16]))

CALLS = {
    "weights": lambda t: ops.paged_attention_weights(t["q1"], t["k"], t["v"], t["table"], t["lens"], t["weights"], block_size=BS),
    "shared": lambda t: ops.paged_attention_shared(t["q1"], t["k"], t["v"], t["table"], t["lens"], CU, PREFIX, block_size=BS),
    "shared with weights": lambda t: ops.paged_attention_shared(t["q1"], t["k"], t["v"], t["table"], t["lens"], CU, PREFIX, block_size=BS, weights=t["weights"]),
    "chunk": lambda t: ops.flash_attention_paged_weights(t["q"], t["k"], t["v"], t["table"], NEW, TOTAL, t["weights"]),
    "evict": lambda t: ops.kv_evict(t["k"], t["v"], t["weights"], t["table"], t["lens"], keep=8, recent=2, first=1),
    "evict by sequence": lambda t: ops.kv_evict(t["k"], t["v"], t["weights"], t["table"], t["lens"], keep=8, recent=2, first=t["first"])}
USES = {"weights": ["q1", "k", "v", "table", "lens", "weights"], "shared": ["q1", "k", "v", "table", "lens"], "shared with weights": ["q1", "k", "v", "table", "lens", "weights"],
        "chunk": ["q", "k", "v", "table", "weights"], "evict": ["k", "v", "weights", "table", "lens"], "evict by sequence": ["k", "v", "weights", "table", "lens", "first"]}


def _tensors(dev):
    half = lambda *shape: torch.zeros(shape, dtype=torch.bfloat16, device=dev)
    ints = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=dev)
    return dict(q=half(9, HQ, D), q1=half(B, HQ, 1, D), k=half(6, BS, HKV, D), v=half(6, BS, HKV, D), table=ints(B, W), lens=ints(B), first=ints(B),
                weights=torch.zeros((B, HKV, W * BS), device=dev))


class Reached(Exception):
    """The call has come to a launch."""


@pytest.fixture
def as_on_device(monkeypatch):
    """Host tensors as if they were on a device, and a launch layer that says that it was reached."""
    class Launch:
        def __getattr__(self, name):
            if name.startswith("sca_launch"):
                def launch(*args):
                    raise Reached(name)
                return launch
            return getattr(_lib.lib(), name)
    monkeypatch.setattr(ops, "_native", lambda: ops._GeneralFormOnly())
    monkeypatch.setattr(ops, "_elsewhere", lambda t, stream: False)
    monkeypatch.setattr(ops, "_stream_ptr", lambda stream=None: 0)
    monkeypatch.setattr(ops, "acquire_scratch_fp32", lambda n, *a, **more: torch.empty(n))
    monkeypatch.setattr(ops, "lib", Launch)
    on_host = []

    def require(*tensors):
        for t in tensors:
            if any(t is x for x in on_host):
                raise _lib.ScaError(5, "device=cpu")
    monkeypatch.setattr(ops, "_require_cuda", require)
    return on_host


@pytest.mark.parametrize("name", CALLS)
def test_calls_on_the_host_are_refused(name):
    with pytest.raises(_lib.ScaError, match="device=cpu"):
        CALLS[name](_tensors("cpu"))


@pytest.mark.parametrize("name", CALLS)
def test_the_same_calls_are_served_on_a_device(as_on_device, name):
    with pytest.raises(Reached):
        CALLS[name](_tensors("cpu"))


@pytest.mark.parametrize("name,tensor", [(n, t) for n in CALLS for t in USES[n]])
def test_a_tensor_on_the_host_is_refused(as_on_device, name, tensor):
    t = _tensors("cpu")
    as_on_device.append(t[tensor])
    with pytest.raises(_lib.ScaError, match="device=cpu"):
        CALLS[name](t)


@pytest.mark.gpu
@pytest.mark.parametrize("name,tensor", [(n, t) for n in CALLS for t in USES[n]])
def test_a_tensor_on_the_host_among_others_on_the_device(name, tensor):
    t = _tensors("cuda")
    CALLS[name](t)
    t[tensor] = t[tensor].cpu()
    with pytest.raises(_lib.ScaError, match="device=cpu"):
        CALLS[name](t)
