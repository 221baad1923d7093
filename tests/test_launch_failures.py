"""A kernel launch that fails half-way through a call leaves the library's state
as it was.  The call's own object code runs on the host against a stand-in for
the CUDA runtime that refuses a chosen launch; nothing reaches a GPU."""
from __future__ import annotations

import ctypes as C
import subprocess

import pytest

from tensorcrate_b200 import _native as N
from tensorcrate_b200 import build

RUNTIME = r"""
#include <cstddef>
struct CUstream_st;
enum cudaError : int { cudaSuccess = 0, cudaErrorLaunchFailure = 719 };
struct dim3 { unsigned x, y, z; };
static int launches, refuse, ticket, error, taken[64];
static dim3 push_grid, push_block;
extern "C" {
void refuse_launch(int n) { launches = error = 0; refuse = n; }
int launch_count() { return launches; }
int ticket_taken(int n) { return taken[n]; }
void **__cudaRegisterFatBinary(void *) { static void *h; return &h; }
void __cudaRegisterFatBinaryEnd(void **) {}
void __cudaUnregisterFatBinary(void **) {}
void __cudaRegisterFunction(void **, const char *, char *, const char *, int, void *, void *, void *, void *, int *) {}
unsigned __cudaPushCallConfiguration(dim3 g, dim3 b, size_t, CUstream_st *) { push_grid = g; push_block = b; return 0; }
cudaError __cudaPopCallConfiguration(dim3 *g, dim3 *b, size_t *s, void *stream) {
  *g = push_grid; *b = push_block; *s = 0; *static_cast<void **>(stream) = nullptr;
  return cudaSuccess;
}
// square_sums(set, partial, slot, ticket, norm)
cudaError cudaLaunchKernel(const void *, dim3, dim3, void **args, size_t, CUstream_st *) {
  const int n = launches++;
  if (n == refuse) { error = cudaErrorLaunchFailure; return cudaErrorLaunchFailure; }
  taken[n] = *static_cast<int **>(args[3]) != nullptr;
  return cudaSuccess;
}
cudaError cudaLaunchKernelExC(const void *, const void *, void **) { return cudaSuccess; }
}
namespace tc {
int fail(int status, const char *, ...) { return status; }
int check_cuda(cudaError e, const char *) { return e; }
int check_launch(const char *) { const int e = error; error = 0; return e; }
int sm_count() { return 148; }
int scratch(size_t, void **out, CUstream_st *) { static double room[1 << 16]; *out = room; return 0; }
int counters(size_t, int **out, CUstream_st *) { *out = &ticket; return 0; }
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    where = tmp_path_factory.mktemp("runtime")
    build.BUILD.mkdir(exist_ok=True)
    objects = [build._compile(build.CSRC / "gradnorm.cu", False, [])]
    (where / "runtime.cpp").write_text(RUNTIME)
    out = where / "lib.so"
    # -Bsymbolic: its own stand-ins, not a runtime that the process has loaded
    subprocess.run(["g++", "-shared", "-fPIC", "-O1", "-Wl,-Bsymbolic", "-o", str(out), str(where / "runtime.cpp"),
                    *map(str, objects)], check=True)
    return C.CDLL(str(out), mode=C.RTLD_LOCAL)


def test_a_failed_launch_of_the_norm_leaves_no_ticket_taken(lib):
    """1100 tensors are three launches.  The stream's counter is shared with
    every kernel that takes tickets, and each sets it back to zero: whichever
    launch fails, none that ran has taken from it."""
    count = 1100
    grads = (N.Gradient * count)()
    for g in grads:
        g.g, g.out, g.n, g.dtype = 0x10000, 0x10000, 100, N.F32
    for refused in range(3):
        lib.refuse_launch(refused)
        assert lib.tc_grad_norm(grads, C.c_size_t(count), C.c_void_p(0x1000), None) != N.OK
        assert lib.launch_count() == refused + 1
        assert not any(lib.ticket_taken(n) for n in range(refused))
    lib.refuse_launch(-1)
    assert lib.tc_grad_norm(grads, C.c_size_t(count), C.c_void_p(0x1000), None) == N.OK
    assert lib.launch_count() == 3
    assert [lib.ticket_taken(n) for n in range(3)] == [0, 0, 1]
