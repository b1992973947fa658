"""How hcu_attention_paged and hcu_prefill_varlen launch their kernels, on the CPU: their host code linked with a stand-in for
the CUDA runtime that records launches and refuses those that it is told to."""
import ctypes
import os
import shutil
import subprocess

import pytest

from hachiue_b200 import _lib, build

FAKE = r"""
#include <cstdarg>
#include <cstring>
#include <vector>
#include "context.h"

struct Launch { unsigned grid[3], block, cluster, dependent; };
static std::vector<Launch> launches;
static int refuse_clusters, refuse_all;
static cudaError_t last = cudaSuccess;

extern "C" {
cudaError_t cudaGetDevice(int* d) { *d = 0; return cudaSuccess; }
cudaError_t cudaSetDevice(int) { return cudaSuccess; }
cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute, int) { return cudaSuccess; }
cudaError_t cudaGetLastError() { cudaError_t e = last; last = cudaSuccess; return e; }
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t* c, const void*, void**) {
  Launch l = {{c->gridDim.x, c->gridDim.y, c->gridDim.z}, c->blockDim.x, 0, 0};
  for (unsigned i = 0; i < c->numAttrs; i++) {
    if (c->attrs[i].id == cudaLaunchAttributeClusterDimension) l.cluster = c->attrs[i].val.clusterDim.x;
    if (c->attrs[i].id == cudaLaunchAttributeProgrammaticStreamSerialization) l.dependent = 1;
  }
  if ((l.cluster && refuse_clusters) || refuse_all) return last = cudaErrorInvalidConfiguration;
  launches.push_back(l);
  return cudaSuccess;
}
cudaError_t cudaLaunchKernel(const void*, dim3 g, dim3 b, void**, size_t, cudaStream_t) {
  if (refuse_all > 1) return last = cudaErrorInvalidConfiguration;
  launches.push_back({{g.x, g.y, g.z}, b.x, 0, 0});
  return cudaSuccess;
}
void** __cudaRegisterFatBinary(void*) { static void* p; return &p; }
void __cudaRegisterFatBinaryEnd(void**) {}
void __cudaUnregisterFatBinary(void**) {}
void __cudaRegisterFunction(void**, const char*, char*, const char*, int, uint3*, uint3*, dim3*, dim3*, int*) {}
unsigned __cudaPushCallConfiguration(dim3, dim3, size_t, void*) { return 0; }
cudaError_t __cudaPopCallConfiguration(dim3* g, dim3* b, size_t* s, void*) { return *g = *b = dim3(1), *s = 0, cudaSuccess; }
}
namespace hcu {
int fail(int code, const char*, ...) { return code; }
int check_cuda(cudaError_t e, const char*) { return e == cudaSuccess ? HCU_OK : HCU_ECUDA; }
int begin_op(hcu_context*, const char*) { return HCU_OK; }
int after_launch(const char* what) { return check_cuda(cudaGetLastError(), what); }
int make_tensor_map(CUtensorMap*, CUtensorMapDataType, int, void*, const uint64_t*, const uint64_t*, const uint32_t*, CUtensorMapSwizzle) {
  return HCU_OK;
}
}
extern "C" int run(const hcu_attention_paged_params* p, const hcu_paged_kv* kv, size_t workspace, int clusters_refused, int all_refused,
                   unsigned (*out)[6], int* n, int* left) {
  hcu_context h;
  h.workspace = (void*)(1 << 20);
  h.workspace_bytes = workspace;
  launches.clear();
  refuse_clusters = clusters_refused, refuse_all = all_refused, last = cudaSuccess;
  const int rc = hcu_attention_paged(&h, p, (void*)4096, kv, (void*)4096);
  *n = (int)launches.size();
  for (int i = 0; i < *n; i++) std::memcpy(out[i], &launches[i], 24);
  *left = last;
  return rc;
}
extern "C" int run_prefill(const hcu_prefill_varlen_params* p, int all_refused, int* n, int* left) {
  hcu_context h;
  h.workspace = (void*)(1 << 20);
  h.workspace_bytes = 64 << 20;
  launches.clear();
  refuse_all = all_refused, last = cudaSuccess;
  const int rc = hcu_prefill_varlen(&h, p, (void*)4096, (void*)4096, (void*)4096, (void*)4096);
  *n = (int)launches.size();
  *left = last;
  return rc;
}
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    if not shutil.which("g++"):
        pytest.skip("no g++")
    build.build()
    objs = []
    for name in ("attention_paged", "prefill_varlen"):
        obj, src = os.path.join(build.BUILD, name + ".o"), os.path.join(build.CSRC, name + ".cu")
        if not os.path.exists(obj) or os.path.getmtime(obj) < os.path.getmtime(src):
            os.makedirs(build.BUILD, exist_ok=True)
            build._compile(src, False, [])
        objs.append(obj)
    d = tmp_path_factory.mktemp("host")
    fake, lib = d / "fake.cpp", d / "host.so"
    fake.write_text(FAKE)
    cuda = os.path.join(os.path.dirname(os.path.dirname(build.nvcc())), "include")
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-Wl,-Bsymbolic", "-I", cuda, "-I", build.INCLUDE, "-I", build.CSRC, str(fake), *objs, "-o", str(lib)],
                   check=True, capture_output=True)
    return ctypes.CDLL(str(lib))


def launches(host, batch=1, H=16, KV=8, D=128, S=1, max_context=1024, workspace=64 << 20, clusters_refused=0, all_refused=0,
             dtype=_lib.DT_F32, window=0):
    p = _lib.hcu_attention_paged_params(batch, S, H, window, dtype, max_context, -(-max_context // 16), 4096, 4096)
    kv = _lib.hcu_paged_kv(_lib.KV_Q4_0, 16, 1000, KV, D, 4096, 4096, 4096, 4096)
    out, n, left = ((ctypes.c_uint * 6) * 8)(), ctypes.c_int(), ctypes.c_int()
    rc = host.run(ctypes.byref(p), ctypes.byref(kv), ctypes.c_size_t(workspace), clusters_refused, all_refused, out, ctypes.byref(n),
                  ctypes.byref(left))
    return rc, [dict(zip(("x", "y", "z", "block", "cluster", "dependent"), row)) for row in list(out)[:n.value]], left.value


def test_short_contexts_take_clusters(host):
    rc, got, left = launches(host)
    assert rc == 0 and left == 0 and len(got) == 1
    assert got[0]["cluster"] > 1 and got[0]["x"] == 8 * got[0]["cluster"] and not got[0]["dependent"]


@pytest.mark.parametrize("case", [dict(), dict(max_context=16), dict(H=32, dtype=_lib.DT_BF16, S=3), dict(D=256, H=16, KV=2, S=4),
                                  dict(batch=7, window=100, max_context=4096)])
def test_a_refused_cluster_falls_back(host, case):
    """Where the device has no room for a cluster the call goes by equal pieces (joined by a second kernel) or, without the
    workspace for that, by whole units, and leaves no error behind for the next call."""
    rc, got, left = launches(host, **case)
    assert rc == 0 and len(got) == 1 and got[0]["cluster"]
    rc, got, left = launches(host, clusters_refused=1, **case)
    assert rc == 0 and left == 0
    assert not got[0]["cluster"] and not got[0]["dependent"] and got[0]["block"] == 256
    assert len(got) == (1 if got[0]["x"] == 1 else 2)
    if len(got) == 2:
        assert got[1]["dependent"] and got[1]["x"] == got[0]["x"] - 1 and got[1]["block"] == 128
    rc, got, left = launches(host, clusters_refused=1, workspace=(1 << 18) + 4096, **case)
    assert rc == 0 and left == 0 and len(got) == 1 and not got[0]["cluster"] and got[0]["x"] <= 296


def test_a_launch_that_fails_is_reported_once(host):
    """By the call that makes it: the error does not stay for a later one to find."""
    for case in (dict(), dict(max_context=100000)):
        rc, got, left = launches(host, all_refused=1, **case)
        assert rc == _lib.HCU_ECUDA and not got and left == 0
    n, left = ctypes.c_int(), ctypes.c_int()
    for total, before in ((64, 0), (100000, 1)):  # in one launch; behind the list of items
        p = _lib.hcu_prefill_varlen_params(2, 16, 8, 128, 0, _lib.DT_BF16, total, total, 4096, None, 0, 0, 0)
        assert host.run_prefill(ctypes.byref(p), 0, ctypes.byref(n), ctypes.byref(left)) == 0 and n.value == before + 1
        for refused in (1, 2):
            assert host.run_prefill(ctypes.byref(p), refused, ctypes.byref(n), ctypes.byref(left)) == _lib.HCU_ECUDA
            assert left.value == 0 and n.value == (before if refused == 1 else 0)
