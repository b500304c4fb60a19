"""Which kernels a call launches, and on how many blocks: the call is recorded into a graph, whose nodes the driver describes."""
import ctypes as C

from rust_ascend_b200.runtime import _check


class _KernelNode(C.Structure):      # CUDA_KERNEL_NODE_PARAMS_v2
    _fields_ = [("func", C.c_void_p), ("grid", C.c_uint * 3), ("block", C.c_uint * 3), ("shared", C.c_uint), ("params", C.c_void_p), ("extra", C.c_void_p),
                ("kern", C.c_void_p), ("ctx", C.c_void_p)]


def launched(client, call):
    """[(kernel's mangled name, blocks)] in the order of recording.  `call` has run once before, and is not run here."""
    cuda = C.CDLL("libcuda.so.1")

    def ok(code):
        assert code == 0, f"CUDA driver status {code}"
    stream = C.c_void_p()
    _check(client._lib.rb_stream(client._ctx, C.byref(stream)))
    found = []
    _check(client._lib.rb_graph_begin(client._ctx))
    try:
        call()
        status, graph, count = C.c_int(), C.c_void_p(), C.c_size_t()
        ok(cuda.cuStreamGetCaptureInfo_v2(stream, C.byref(status), None, C.byref(graph), None, None))
        ok(cuda.cuGraphGetNodes(graph, None, C.byref(count)))
        nodes = (C.c_void_p * count.value)()
        ok(cuda.cuGraphGetNodes(graph, nodes, C.byref(count)))
        for node in nodes:
            kind, p, name = C.c_int(), _KernelNode(), C.c_char_p()
            ok(cuda.cuGraphNodeGetType(C.c_void_p(node), C.byref(kind)))
            if kind.value != 0:      # CU_GRAPH_NODE_TYPE_KERNEL
                continue
            ok(cuda.cuGraphKernelNodeGetParams_v2(C.c_void_p(node), C.byref(p)))
            ok(cuda.cuKernelGetName(C.byref(name), C.c_void_p(p.kern)) if p.kern else cuda.cuFuncGetName(C.byref(name), C.c_void_p(p.func)))
            found.append((name.value.decode(), p.grid[0] * p.grid[1] * p.grid[2]))
    finally:
        g = C.c_uint64()
        _check(client._lib.rb_graph_end(client._ctx, C.byref(g)))
        _check(client._lib.rb_graph_destroy(client._ctx, g))
    return found
