"""The build is reproducible: the same source gives the same bytes wherever its objects lie."""
import subprocess

SOURCE = """#include <hip/hip_runtime.h>
static __device__ int counter;
__global__ void k(float* p) { p[threadIdx.x] = threadIdx.x + counter; }
extern "C" void go(float* p) { k<<<1, 64>>>(p); }
"""


def test_objects_do_not_depend_on_their_folder(tmp_path):
    from psgd_torch_amd import build
    src = tmp_path / "unit.hip"
    src.write_text(SOURCE)
    objs = []
    for d in ("one", "another"):
        (tmp_path / d).mkdir()
        obj = tmp_path / d / "unit.o"
        subprocess.run(build.object_command("/opt/rocm/bin/hipcc", str(src), str(obj)), check=True, capture_output=True)
        objs.append(obj.read_bytes())
    assert objs[0] == objs[1]
