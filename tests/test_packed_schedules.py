"""The warp roles of the packed kernels under adversarial schedules, on the CPU: test_barrier_schedules.py's simulator (its
sources as they are) with another main."""

import shutil
import subprocess
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent
CSRC = HERE.parent / "flash_attention_triton_b200" / "csrc"

# What the packed kernels use beyond the others: one lane stands for a warp, a CTA of a cluster meets nobody.
STAND_INS = """
struct int4 { int x, y, z, w; };
inline int4 make_int4(int x, int y, int z, int w) { return {x, y, z, w}; }
inline float4 make_float4(float x, float y, float z, float w) { return {x, y, z, w}; }
enum { cudaLaunchAttributeClusterDimension = 100 };
inline unsigned __reduce_add_sync(unsigned, unsigned x) { return x; }
template <typename T> T __shfl_sync(unsigned, T x, int) { return x; }
template <typename T> T __shfl_up_sync(unsigned, T x, int) { return x; }
inline unsigned __ballot_sync(unsigned, bool x) { return x; }
inline int __ffs(unsigned x) { return __builtin_ffs(x); }
inline int __popc(unsigned x) { return __builtin_popcount(x); }
namespace fa2 {
inline uint32_t cluster_address(uint32_t a, uint32_t) { return a; }
FA2_NOTHING(cluster_sync) FA2_NOTHING(st_cluster_v4)
inline void grid_wait_unless(const unsigned*) { sim_wait_previous(); }
FA2_NOTHING(release_flag)
}
"""


@pytest.fixture(scope="module")
def simulator(tmp_path_factory):
    build = tmp_path_factory.mktemp("packed_schedules")
    for name in ("common.cuh", "mma_issue.cuh", "bwd_roles.cuh", "packed.cuh", "paged.cuh", "packed_fwd.cu", "packed_bwd.cu"):
        shutil.copy(CSRC / name, build)
    header = (HERE / "schedules" / "cuda_runtime.h").read_text()
    field = "struct { int programmaticStreamSerializationAllowed; } val;"
    assert header.count(field) == 1
    header = header.replace(field, "struct { int programmaticStreamSerializationAllowed; struct { unsigned x, y, z; } clusterDim; } val;")
    (build / "cuda_runtime.h").write_text(header + STAND_INS)
    for stand_in in ("cuda.h", "ptx.cuh"):
        (build / stand_in).write_text('#include "cuda_runtime.h"\n')
    main = (HERE / "schedules" / "main.cpp").read_text()
    assert main.count('#include "bwd.cu"') == 1
    main = main[: main.index('#include "bwd.cu"')] + (HERE / "schedules_packed" / "main_packed.inc").read_text()
    (build / "main.cpp").write_text(main)
    subprocess.run(["g++", "-std=c++17", "-O1", "-w", "-D__CUDACC__", "-I.", "main.cpp", "-o", "simulator"], cwd=build, check=True,
                   capture_output=True, text=True)
    return build / "simulator"


def run(simulator, kernel, d, heads, kv_heads, lengths, step=128, cluster=1, sms=2, schedules=40, giveup=False):
    a = [kernel, d, heads, kv_heads, step, cluster, sms, schedules, int(giveup), *lengths]
    done = subprocess.run([simulator, *map(str, a)], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, (a, done.stdout + done.stderr)


LENGTHS = [[1], [128], [129, 700, 3], [449, 640, 128, 1]]


@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("heads,kv_heads", [(2, 1), (3, 1), (2, 2)])
def test_forward(simulator, d, heads, kv_heads, lengths):
    for sms in (1, 3, 64):  # one CTA takes every item; some take several; each has one (and reads cu_seqlens itself)
        if sms < 64 or len(lengths) == 1:  # one lane stands for a warp, and it knows one sequence
            run(simulator, "fwd", d, heads, kv_heads, lengths, sms=sms)


@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("d,step", [(32, 64), (32, 128), (64, 64), (64, 128), (96, 128), (128, 128)])
def test_backward(simulator, d, step, lengths):
    for cluster in (1, 2, 4):
        run(simulator, "dkdv", d, 2 * max(2, cluster), 2, lengths, step, cluster)
    run(simulator, "dkdv", d, 3, 1, lengths, step)
    run(simulator, "dq", d, 3, 1, lengths, step)


@pytest.mark.parametrize("kernel,d,step", [("fwd", 64, 128), ("fwd", 128, 128), ("dkdv", 64, 64), ("dkdv", 64, 128), ("dkdv", 128, 128),
                                           ("dq", 64, 64), ("dq", 64, 128), ("dq", 128, 128)])
def test_that_gives_up_a_wait(simulator, kernel, d, step):
    """Whichever wait runs into its limit, every CTA ends."""
    for lengths in ([128], [300, 640]):
        for cluster in (1, 2) if kernel == "dkdv" else (1,):
            run(simulator, kernel, d, 2, 1, lengths, step, cluster, giveup=True)
