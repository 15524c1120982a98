"""Which kernels a call launches, read from a graph that it is captured into: tests of a form that a rule chooses say that it was the one that ran."""
import ctypes as C

PREFIX, OWN, FINISH, ONE, CHUNK = "flash_fwd_sm100_kernel", "decode_own_kernel", "decode_finish_kernel", "decode_step_cluster_kernel", "chunk_weights_kernel"
THREE = [PREFIX, OWN, FINISH]  # a decode over shared prefixes that fills the machine
TWO = [OWN, FINISH]            # one without a shared page
ALL = (PREFIX, OWN, FINISH, ONE, CHUNK)

KERNEL_NODE = 0


class KernelNodeParams(C.Structure):  # CUDA_KERNEL_NODE_PARAMS of cuda.h
    _fields_ = [("func", C.c_void_p)] + [(n, C.c_uint) for n in ("grid_x", "grid_y", "grid_z", "block_x", "block_y", "block_z", "shared_bytes")] + \
        [(n, C.c_void_p) for n in ("params", "extra", "kern", "ctx")]


def _ask(result):
    assert result == 0, f"CUDA driver: error {result}"


def launches(call):
    """Those of ALL that `call` launches, in their order."""
    import torch
    call()  # what a first call sets up is not for a capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    driver, handle, count = C.CDLL("libcuda.so.1"), C.c_void_p(graph.raw_cuda_graph()), C.c_size_t()
    _ask(driver.cuGraphGetNodes(handle, None, C.byref(count)))
    nodes = (C.c_void_p * count.value)()
    _ask(driver.cuGraphGetNodes(handle, nodes, C.byref(count)))
    found = []
    for node in nodes:
        kind, params, name = C.c_int(), KernelNodeParams(), C.c_char_p()
        _ask(driver.cuGraphNodeGetType(C.c_void_p(node), C.byref(kind)))
        if kind.value != KERNEL_NODE:
            continue
        _ask(driver.cuGraphKernelNodeGetParams_v2(C.c_void_p(node), C.byref(params)))
        if params.func:
            _ask(driver.cuFuncGetName(C.byref(name), C.c_void_p(params.func)))
        else:
            _ask(driver.cuKernelGetName(C.byref(name), C.c_void_p(params.kern)))
        found += [kernel for kernel in ALL if kernel.encode() in name.value]
    return found
