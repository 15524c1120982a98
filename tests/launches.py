"""Which kernels a call launches, read from a trace: tests of a form that a rule chooses say that it was the one that ran."""
import json

import pytest

PREFIX, OWN, FINISH, ONE, CHUNK = "flash_fwd_sm100_kernel", "decode_own_kernel", "decode_finish_kernel", "decode_step_cluster_kernel", "chunk_weights_kernel"
THREE = [PREFIX, OWN, FINISH]  # a decode over shared prefixes that fills the machine
TWO = [OWN, FINISH]            # one without a shared page


def launches(call, path):
    """This library's kernels that `call` launches, in the order of their start. `path`: a folder for the trace."""
    import torch
    call()
    torch.cuda.synchronize()
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
        call()
        torch.cuda.synchronize()
    trace = path / "trace.json"
    prof.export_chrome_trace(str(trace))
    kernels = [e for e in json.load(open(trace))["traceEvents"] if e.get("cat") == "kernel"]
    if not kernels:
        pytest.skip("launches cannot be traced here")
    return [e["name"].split("sca_b200::")[1].split("(anonymous namespace)::")[-1].split("flash::")[-1].split("<")[0].split("(")[0]
            for e in sorted(kernels, key=lambda e: e["ts"]) if "sca_b200::" in e["name"]]
