"""What the kernels' entry points refuse on the host, before anything is launched: no device is needed."""
import subprocess
import sys

BAD_SIZE = -3

CODE = """
from camelid_b200.csrc import ops
f = ops._fn("gemm_few", "cml_gemm_few")
for splits in {splits}:
    print(f(4096, 64, 1, 4096, 64, 16, {k}, 4096, 16, ops.FEW_F32, None, 0, None, 0, 0, 0.0, None, 0, None, 0, None, splits, 0, None, None))
"""


def _codes(k, splits):
    out = subprocess.run([sys.executable, "-c", CODE.format(k=k, splits=splits)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr
    return [int(line) for line in out.stdout.split() if line.lstrip("-").isdigit()]


def test_shares_of_k_that_do_not_cut_it():
    """No shares, fewer than none, empty ones, and ones of more columns than a block takes (a child process: it may die of it)."""
    assert _codes(4096, [0, -1, 1, 9]) == [BAD_SIZE] * 4


DEVICES = r"""
#include <cuda_runtime.h>
#include <stdio.h>
static int device = 0, asked = 0, read = 0;
static cudaError_t fake_device(int* d) { *d = device; return device < 0 ? cudaErrorNoDevice : cudaSuccess; }
template <typename K> static cudaError_t fake_set(K, cudaFuncAttribute, int) { ++asked; return cudaSuccess; }
static cudaError_t fake_read(int* v, cudaDeviceAttr, int dev) { ++read; *v = dev == 0 ? 148 : 132; return cudaSuccess; }
#define cudaGetDevice fake_device
#define cudaFuncSetAttribute fake_set
#define cudaDeviceGetAttribute fake_read
#include "common.cuh"
__global__ void kernel(int) {}
int main() {
    const int devices[] = {0, 0, 1, 1, 0, 40, 40, -1};
    for (int d : devices) {
        device = d, asked = 0, read = 0;
        const int sms = (cml_sm_count(), cml_sm_count());
        cml_allow_smem<kernel>(100000);
        cml_allow_smem<kernel>(90000);
        cml_allow_wide_clusters<kernel>();
        cml_allow_wide_clusters<kernel>();
        printf("%d %d %d ", sms, read, asked);
    }
    return 0;
}
"""


def test_what_is_set_once_is_set_once_a_device(tmp_path):
    """Limits of shared memory and clusters, and the number of multiprocessors, belong to the current device: the second device's first
    call sets and reads its own. (Host code alone, with the runtime's calls replaced.)"""
    from camelid_b200.csrc import build
    source, program = tmp_path / "devices.cu", tmp_path / "devices"
    source.write_text(DEVICES)
    flags = [f for f in build.NVCC_FLAGS if f not in ("--shared",)]
    subprocess.run([build.find_nvcc(), *flags, "-I", build.CSRC_DIR, "-o", str(program), str(source)], check=True, timeout=600)
    out = [int(x) for x in subprocess.run([str(program)], capture_output=True, text=True, check=True, timeout=60).stdout.split()]
    known = {0: [(148, 1, 2), (148, 0, 0), (148, 0, 0)], 1: [(132, 1, 2), (132, 0, 0)]}
    want = [known[0][0], known[0][1], known[1][0], known[1][1], known[0][2], (148, 0, 4), (148, 0, 4), (148, 0, 4)]      # 40 and none: not remembered
    assert [tuple(out[i:i + 3]) for i in range(0, len(out), 3)] == want
