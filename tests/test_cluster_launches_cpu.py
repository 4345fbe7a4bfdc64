"""CPU tier: what keeps the clusters' unbounded waits (tensor-memory allocation, cluster barriers) from waiting on one another, read from
the launches against the stand-in runtime (fake_cudart.c) in a process of its own, this file as the program."""
import ctypes
import glob
import os
import re

from test_feed_forward_launches_cpu import _run as run_check
from test_launches_cpu import LAUNCH, ROOT, Runtime

import test_feed_forward_launches_cpu as launches

i64, i32 = ctypes.c_int64, ctypes.c_int
SM_SMEM, CTA_RESERVED = 233472, 1024                  # shared memory of an SM, and what the system takes of it per CTA
CLUSTERS = """
cudaError_t cudaOccupancyMaxActiveClusters(int* n, const void* fn, const cudaLaunchConfig_t* c) {
    (void)fn;
    *n = 148 / (int)c->attrs[0].val.clusterDim.x;
    return cudaSuccess;
}
"""


def check_clusters_have_their_sms_alone():
    """A CTA of a cluster holds its tensor memory while it waits for the others of its cluster, so none of them may wait for that memory
    behind another: no two CTAs of cluster launches fit on one SM."""
    rt = Runtime()
    P = rt.p(9)
    seen, limit = [], {}
    cb = LAUNCH(lambda name, grid, block, smem, cluster, early, args: seen.append((name.decode(), smem, cluster)) or 0)
    rt.fake.fake_callbacks(cb, *rt._keep[1:])
    rt.on_limit = lambda name, value: limit.__setitem__(name, value) or 0
    clusters = set()

    def run(call, what):
        seen.clear()
        assert call() == 0, (what, rt.lib.hkb_last_error())
        for name, smem, cluster in seen:
            if cluster > 1:
                clusters.add(name)
                assert 2 * (smem + CTA_RESERVED) > SM_SMEM, (what, name, smem, cluster)
                assert smem <= limit[name], (what, name, smem, limit[name])

    for K in (128, 256, 1024, 2048, 4096, 8192, 14336):
        for M in (*range(1, 10), 16, 17, 32, 33, 64, 65, 128, 300):
            for N in (*range(16, 513, 16), 1024, 1032, 4096):
                for batch in (1, 2):
                    run(lambda: rt.lib.hkb_gemm_fp8_pts_epilogue(*P[:5], P[5], i32(2), P[6], i64(batch), i64(M), i64(N), i64(K), None), ("token", batch, M, N, K))
                if N % 128 == 0:
                    run(lambda: rt.lib.hkb_gemm_fp8_blockscale_epilogue(*P[:5], i64(128), P[5], i32(2), P[6], i64(M), i64(N), i64(K), None), ("block", M, N, K))
                    for fp8 in (False, True):
                        run(lambda: rt.lib.hkb_gemm_fp8_blockscale_gated(P[0], P[1], P[2], P[3] if fp8 else None, P[4], P[5], i32(4), P[6], i64(M), i64(N), i64(K), None),
                            ("gated", M, N, K, fp8))
    for what, call in rt.calls().items():
        run(call, what)
    assert any("gemm_fp8_skinny_kernel" in n for n in clusters) and any("blockscale_skinny" in n for n in clusters) and len(clusters) >= 12, clusters


def test_clusters_have_their_sms_alone(tmp_path, monkeypatch):
    monkeypatch.setattr(launches, "__file__", __file__)
    run_check("check_clusters_have_their_sms_alone", tmp_path, CLUSTERS)


def test_no_dependent_launch_before_the_tensor_memory_is_there():
    """A kernel that lets the next launch start (whose CTAs allocate tensor memory and then wait for this one to end) has its own by
    then: in the source, a CTA barrier lies between the allocation and the trigger."""
    both = 0
    for path in sorted(glob.glob(os.path.join(ROOT, "amd-kernels_b200", "csrc", "*.cu"))):
        with open(path) as f:
            code = re.sub(r"//[^\n]*", "", f.read())
        for body in code.split("__global__")[1:]:
            alloc, trigger = body.find("tmem_alloc"), body.find("pdl_trigger()")
            if alloc >= 0 and trigger >= 0:
                both += 1
                assert 0 <= body.find("__syncthreads()", alloc) < trigger, (os.path.basename(path), body[:120])
    assert both == 3


if __name__ == "__main__":
    import sys
    globals()[sys.argv[1]]()
