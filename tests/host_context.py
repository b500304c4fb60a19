"""A ComputeClient whose context has no device (tests/host_model/context_host.cpp): for calls that have to be refused."""
import ctypes as C
import os
import subprocess

from rust_ascend_b200 import TensorBuffer, _lib, build
from rust_ascend_b200.runtime import ComputeClient

HERE = os.path.dirname(os.path.abspath(__file__))


class HostClient(ComputeClient):
    """`tensor` registers a storage of exactly the needed bytes at an address that nothing ever reads."""

    def __init__(self, directory):
        build.build()
        library = os.path.join(directory, "context_host.so")
        cuda = os.path.join(os.path.dirname(os.path.dirname(build.NVCC)), "include")
        subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", build.CSRC, "-I", os.path.join(build.ROOT, "include"), "-I", cuda, "-x", "c++",
                        os.path.join(HERE, "host_model", "context_host.cpp"), "-o", library], check=True)
        self._host = C.CDLL(library)
        self._host.host_context.restype = C.c_void_p
        super().__init__(C.c_void_p(self._host.host_context()), None)
        self._next = 1 << 40

    def storage(self, nbytes, misalign=0):
        at = self._next + misalign
        self._next += (nbytes + 0xFFFF) & ~0xFFFF | 0x10000
        return self.import_pointer(at, nbytes)

    def tensor(self, shape, dtype, strides=None, offset=0, nbytes=None):
        t = TensorBuffer(0, shape, dtype, strides, offset)
        t.handle = self.storage(max(t.nbytes + offset, 1) if nbytes is None else nbytes)
        return t

    def close(self):
        self._host.host_context_free(self._ctx)
