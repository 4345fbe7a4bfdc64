"""CPU tier: which kernels and grids the feed-forward operators' calls come to, against the stand-in runtime (fake_cudart.c) in a
process of its own, this file as the program.  Torch is not imported: its kernels would register with the stand-in first."""
import ctypes
import os
import shutil
import subprocess
import sys

from test_launches_cpu import HKB_ERR_CUDA, LAUNCH, ROOT, Runtime

i64, f32, i32 = ctypes.c_int64, ctypes.c_float, ctypes.c_int


def check_launches():
    rt = Runtime()
    rt.lib.hkb_gemm_fp8_blockscale_gated_workspace.restype = i64
    P = rt.p(8)

    def launches(call, expect=0):
        seen = []
        rt.on_launch = lambda name, grid, smem, args: seen.append((name, grid, smem)) or 0
        assert call() == expect, rt.lib.hkb_last_error()
        return seen

    def norm(M, D, group):
        return lambda: rt.lib.hkb_add_rmsnorm_quant_fp8(*P[:6], i64(M), i64(D), i64(group), f32(1e-6), None)

    def gated(M, F, K, fp8):
        return lambda: rt.lib.hkb_gemm_fp8_blockscale_gated(P[0], P[1], P[2], P[3] if fp8 else None, P[4], P[5], i32(4), P[6], i64(M), i64(F), i64(K), None)

    # every row has its threads: a team of warps per row, `nw` chunks of `el` elements per thread, as many rows per CTA as teams
    seen = []
    with_block = LAUNCH(lambda name, grid, block, smem, cluster, early, args: seen.append((name.decode(), grid, block)) or 0)
    rt.fake.fake_callbacks(with_block, *rt._keep[1:])
    for M in (1, 2, 3, 147, 148, 149, 1000, 16384, 2147483647):
        for D in (8, 128, 136, 512, 1024, 1032, 2048, 4096, 4104, 5120, 8192, 16384, 16392, 32760, 32768):
            for group in {D, 128 if D % 128 == 0 else D}:
                seen.clear()
                assert norm(M, D, group)() == 0, rt.lib.hkb_last_error()
                (name, grid, block), = seen
                el, nw = (int(v) for v in name.split("add_rmsnorm_quant_kernelILi")[1].split("ELb")[0].split("ELi"))
                assert el == (16 if D % 16 == 0 else 8)
                chunks = D // el
                warps = -(-(-(-chunks // 32)) // nw)
                teams = max(1, 8 // warps)
                assert warps <= 16 and block == 32 * warps * teams, (M, D, name, block)
                assert grid == -(-M // teams), (M, D, name, grid)
    rt.fake.fake_callbacks(*rt._keep)
    # gated: one launch, and a second one for a decode call's codes; shared memory within the limit
    for F, K in ((128, 128), (1152, 4224), (14336, 4096), (28672, 8192)):
        for M in (1, 16, 17, 32, 33, 128, 129, 4096):
            for fp8 in (False, True):
                seen = launches(gated(M, F, K, fp8))
                assert len(seen) == (2 if fp8 and M <= 32 else 1), (M, F, K, fp8, seen)
                assert all(smem <= 232448 for _, _, smem in seen)
                assert seen[0][1] <= 148
                if len(seen) == 2:
                    assert seen[1][1] * 32 >= M * F // 128
    # a failing launch is that call's error and leaves nothing pending
    for call in (norm(4, 512, 128), gated(4, 256, 256, True), gated(300, 256, 256, True)):
        rt.on_launch = lambda *_: 701
        assert call() == HKB_ERR_CUDA and rt.fake.fake_pending() == 0
        rt.on_launch = lambda *_: 0
        assert call() == 0


def check_splits():
    """With clusters to be had (the stand-in says 148 / size at once): every split launch is whole clusters that fit together, at most one
    tile each, and whole waves followed by a split rest add up to the problem's tiles."""
    rt = Runtime()
    rt.lib.hkb_gemm_fp8_blockscale_gated_workspace.restype = i64
    P = rt.p(9)
    seen = []
    cb = LAUNCH(lambda name, grid, block, smem, cluster, early, args: seen.append((name.decode(), grid, smem, cluster)) or 0)
    rt.fake.fake_callbacks(cb, *rt._keep[1:])
    rt.lib.hkb_last_kernel.restype = ctypes.c_char_p
    kinds = {}

    def run(call, what, tiles):
        seen.clear()
        assert call() == 0, (what, rt.lib.hkb_last_error())
        gemms = [x for x in seen if "quant_f32" not in x[0]]
        kinds.setdefault((rt.lib.hkb_last_kernel().decode(), len(gemms)), what)
        for name, grid, smem, cluster in gemms:
            assert smem <= 232448
            if cluster > 1:
                assert grid % cluster == 0 and grid <= 148, (what, name, grid, cluster)
        if len(gemms) == 2:                                     # whole waves, then one cluster per remaining tile
            (_, g0, _, c0), (_, g1, _, c1) = gemms
            assert c0 == 0 and g0 == 148 and c1 in (2, 4, 8) and g1 // c1 in {t % 148 for t in tiles}, (what, gemms)

    for M in (1, 16, 17, 33, 64, 128, 129, 300, 512, 1000, 2048, 4096):
        for N, K in ((128, 128), (128, 8192), (1024, 8192), (1152, 4224), (4096, 2048), (4096, 14336), (14336, 4096), (2048, 8192)):
            m = -(-M // 128)
            run(lambda: rt.lib.hkb_gemm_fp8_blockscale_epilogue(*P[:5], i64(128), P[5], i32(2), P[6], i64(M), i64(N), i64(K), None),
                ("block", M, N, K), (m * (N // 128), m * (N // 256)))
            for fp8 in (False, True):
                run(lambda: rt.lib.hkb_gemm_fp8_blockscale_gated(P[0], P[1], P[2], P[3] if fp8 else None, P[4], P[5], i32(4), P[6], i64(M), i64(N), i64(K), None),
                    ("gated", M, N, K, fp8), (m * (N // 128), m * (N // 64)))
            for batch in (1, 3):
                run(lambda: rt.lib.hkb_gemm_fp8_pts_epilogue(*P[:5], P[5], i32(2), P[6], i64(batch), i64(M), i64(N), i64(K), None), ("token", batch, M, N, K), ())
    split = {k for k, _ in kinds if "split" in k}
    assert len(split) == 9, split                               # three decode kernels; two widths each of block-scale, gated and per-token tiles
    assert any(n == 2 for _, n in kinds)


def _run(check, tmp_path, more=""):
    import pytest
    inc = "/usr/local/cuda/include"
    gcc = shutil.which("gcc")
    if gcc is None or not os.path.exists(os.path.join(inc, "cuda_runtime_api.h")):
        pytest.skip("no C compiler or CUDA runtime headers")
    so, src = str(tmp_path / "fake_cudart.so"), str(tmp_path / "fake.c")
    with open(os.path.join(ROOT, "tests", "fake_cudart.c")) as f, open(src, "w") as g:
        g.write(f.read() + more)
    subprocess.run([gcc, "-std=gnu11", "-O1", "-shared", "-fPIC", "-I", inc, src, "-o", so], check=True, capture_output=True, text=True)
    r = subprocess.run([sys.executable, os.path.abspath(__file__), check], env={**os.environ, "LD_PRELOAD": so}, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr


def test_launches(tmp_path):
    _run("check_launches", tmp_path)


def test_splits(tmp_path):
    _run("check_splits", tmp_path, """
cudaError_t cudaOccupancyMaxActiveClusters(int* n, const void* fn, const cudaLaunchConfig_t* c) {
    (void)fn;
    *n = 148 / (int)c->attrs[0].val.clusterDim.x;
    return cudaSuccess;
}
""")


if __name__ == "__main__":
    globals()[sys.argv[1]]()
