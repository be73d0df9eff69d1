"""Which kernels a call launches, read from a captured graph of it (a profiler may lose events late in a long process)."""
import ctypes
import re

import torch


class _KernelNode(ctypes.Structure):  # (CUDA_KERNEL_NODE_PARAMS, with room behind it)
    _fields_ = [("func", ctypes.c_void_p), ("shape", ctypes.c_uint * 7), ("params", ctypes.c_void_p), ("extra", ctypes.c_void_p),
                ("kern", ctypes.c_void_p), ("context", ctypes.c_void_p), ("room", ctypes.c_void_p * 8)]


def _readable(mangled):
    """``name<whole numbers and truth values of the template>``."""
    m = re.search(r"\d([a-z][a-z_]*_kernel)(I\w*?Ev)?", mangled)
    if m is None:
        return mangled
    values = re.findall(r"L([bi])(\d+)E", m.group(2) or "")
    return m.group(1) + ("<" + ", ".join(("false", "true")[int(v)] if kind == "b" else v for kind, v in values) + ">" if values else "")


def kernels(call):
    """Their names, with the template's numbers; ``call`` has to be one that may be captured."""
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    cuda, handle, count = ctypes.CDLL("libcuda.so.1"), ctypes.c_void_p(graph.raw_cuda_graph()), ctypes.c_size_t()
    assert cuda.cuGraphGetNodes(handle, None, ctypes.byref(count)) == 0
    nodes = (ctypes.c_void_p * count.value)()
    assert cuda.cuGraphGetNodes(handle, nodes, ctypes.byref(count)) == 0
    found = set()
    for node in map(ctypes.c_void_p, nodes):
        kind, of, name = ctypes.c_int(), _KernelNode(), ctypes.c_char_p()
        assert cuda.cuGraphNodeGetType(node, ctypes.byref(kind)) == 0
        if kind.value == 0:  # a kernel
            assert cuda.cuGraphKernelNodeGetParams_v2(node, ctypes.byref(of)) == 0
            assert cuda.cuFuncGetName(ctypes.byref(name), ctypes.c_void_p(of.func)) == 0
            found.add(_readable(name.value.decode()))
    return found


def sm_count():
    return torch.cuda.get_device_properties(0).multi_processor_count
