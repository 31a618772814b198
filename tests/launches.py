"""Which kernels a call launches: their names and grids, from a captured graph of it."""
import ctypes

import torch


class _Kernel(ctypes.Structure):  # CUDA_KERNEL_NODE_PARAMS
    _fields_ = [("func", ctypes.c_void_p), ("grid", ctypes.c_uint * 3), ("block", ctypes.c_uint * 3), ("shared", ctypes.c_uint),
                ("params", ctypes.c_void_p), ("extra", ctypes.c_void_p), ("kern", ctypes.c_void_p), ("ctx", ctypes.c_void_p)]


def launches(call):
    """[(name, CTAs)] of what `call`, given a stream's address, enqueues; it runs once before."""
    call(torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call(torch.cuda.current_stream().cuda_stream)
    cuda = ctypes.CDLL("libcuda.so.1")

    def check(code):
        assert code == 0, code
    raw, count = ctypes.c_void_p(graph.raw_cuda_graph()), ctypes.c_size_t()
    check(cuda.cuGraphGetNodes(raw, None, ctypes.byref(count)))
    nodes = (ctypes.c_void_p * count.value)()
    check(cuda.cuGraphGetNodes(raw, nodes, ctypes.byref(count)))
    found = []
    for node in nodes:
        kind, k, name = ctypes.c_int(), _Kernel(), ctypes.c_char_p()
        check(cuda.cuGraphNodeGetType(ctypes.c_void_p(node), ctypes.byref(kind)))
        if kind.value:  # not a kernel
            continue
        check(cuda.cuGraphKernelNodeGetParams_v2(ctypes.c_void_p(node), ctypes.byref(k)))
        if k.kern:
            check(cuda.cuKernelGetName(ctypes.byref(name), ctypes.c_void_p(k.kern)))
        else:
            check(cuda.cuFuncGetName(ctypes.byref(name), ctypes.c_void_p(k.func)))
        found.append((name.value.decode(), k.grid[0] * k.grid[1] * k.grid[2]))
    return found
