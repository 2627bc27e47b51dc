"""CPU: the workspace of the orthogonalisation is a function of the call's arguments alone. The
size is asked for (and kept) before the library has looked at a device, so a layout that followed
the device's number of SMs could be larger than the workspace that was asked for.

The host code of csrc/lin_ortho.cu is compiled here with its neighbours replaced, among them the
number of SMs."""

import subprocess

import pytest

from linalg_kernels_b200 import build

HARNESS = r"""
#include "CSRC/lin_ortho.cu"
#include <stdio.h>
#include <stdlib.h>

static int g_fake_sms = 148;
namespace chol {
void note_launch(cudaStream_t) {}
int prepare_device_checked(int) { return CHOL_ERR_DEVICE; }
int* device_status_ptr() { return nullptr; }
}
namespace lin {
int sm_count() { return g_fake_sms; }
void use_sm_count(int) {}
int launch_product(const Product&, cudaStream_t) { return CHOL_ERR_DEVICE; }
cudaError_t prepare_products() { return cudaErrorUnknown; }
cudaError_t prepare_small_ortho() { return cudaErrorUnknown; }
cudaError_t prepare_mid_ortho() { return cudaErrorUnknown; }
cudaError_t prepare_few() { return cudaErrorUnknown; }
bool small_supported(int64_t, int64_t, bool) { return false; }
bool mid_supported(int64_t, int64_t, bool) { return false; }
int launch_small(const linalg_matrix*, const linalg_matrix*, const linalg_matrix*, int64_t, int64_t,
                 int64_t, double, int, float, float, int, const float*, float, bool, cudaStream_t) {
  return CHOL_ERR_DEVICE;
}
int launch_mid_ortho(const linalg_matrix*, const linalg_matrix*, const linalg_matrix*, int64_t,
                     int64_t, int64_t, double, int, float, float, int, const float*, float,
                     cudaStream_t) {
  return CHOL_ERR_DEVICE;
}
}
int main() {
  const long sizes[][3] = {{1, 300, 260}, {1, 8192, 8192}, {16, 2048, 2048}, {640, 512, 512},
                           {1, 16384, 28672}, {100000, 130, 300}, {1, 5000, 4096}};
  const int sms[] = {148, 64, 132, 152, 160, 192};
  for (const auto& s : sizes)
    for (int precision = 1; precision <= 2; ++precision) {
      g_fake_sms = 148;
      const size_t want = linalg_orthogonalize_workspace(s[0], s[1], s[2], precision);
      for (int n : sms) {
        g_fake_sms = n;
        const size_t got = linalg_orthogonalize_workspace(s[0], s[1], s[2], precision);
        if (want == 0 || got != want) {
          printf("%ld x %ld x %ld, %d SMs: %zu, not %zu\n", s[0], s[1], s[2], n, got, want);
          return 1;
        }
      }
    }
  puts("ok");
  return 0;
}
"""


def test_workspace_does_not_depend_on_the_device(tmp_path):
    try:
        nvcc = build._nvcc()
    except RuntimeError:
        pytest.skip("no nvcc")
    source, program = tmp_path / "workspace.cu", tmp_path / "workspace"
    source.write_text(HARNESS.replace("CSRC", str(build.CSRC)))
    # no device code is run: unoptimised, host and device
    subprocess.run([nvcc, *build.ARCH_FLAGS, "-std=c++17", "-O0", "-Xptxas", "-O0",
                    "--expt-relaxed-constexpr", "-o", str(program), str(source)], check=True)
    out = subprocess.run([str(program)], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout
