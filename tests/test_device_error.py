"""tl_device_error reads and clears every error word, whichever of them are set (CPU: ops.cu with the readers faked)."""

import shutil
import subprocess

import pytest

from conftest import PKG_DIR, ROOT

NAMES = ("tc", "attn", "decode1", "tp", "paged_attn", "logprob")

# arguments: the six words and the reader that fails (-1: none); prints the status of two calls, the words after each
FAKES = """
#include <cstdio>
#include <cstdlib>
#include <cuda_runtime.h>
#include "tl_api.h"
unsigned int word[6];
int failing;
extern "C" cudaError_t fake_synchronize() { return cudaSuccess; }
namespace tl {
static cudaError_t take(int i, unsigned int* code) {
  if (failing == i) return cudaErrorUnknown;
  *code = word[i];
  word[i] = 0;
  return cudaSuccess;
}
""" + "".join(f"cudaError_t {n}_read_error(unsigned int* code) {{ return take({i}, code); }}\n"
              for i, n in enumerate(NAMES)) + """}
int main(int, char** argv) {
  for (int i = 0; i < 6; ++i) word[i] = atoi(argv[1 + i]);
  failing = atoi(argv[7]);
  for (int n = 0; n < 2; ++n) {
    printf("%d", static_cast<int>(tl_device_error()));
    for (unsigned int w : word) printf(" %u", w);
    printf("\\n");
  }
}
"""


@pytest.fixture(scope="module")
def call(tmp_path_factory):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    home = tmp_path_factory.mktemp("device_error")
    (home / "fakes.cu").write_text(FAKES)
    # what ops.cu launches is not there: nothing here calls it
    cmd = [nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-diag-suppress", "128", "-I",
           str(ROOT / "include"), "-DcudaDeviceSynchronize=fake_synchronize", "-Xlinker",
           "--unresolved-symbols=ignore-all", str(PKG_DIR / "csrc" / "ops.cu"), str(home / "fakes.cu"), "-o",
           str(home / "fakes")]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr

    def run(words, failing=-1):
        r = subprocess.run([str(home / "fakes"), *map(str, words), str(failing)], capture_output=True, text=True)
        assert r.returncode == 0, r.stderr
        return [[int(x) for x in line.split()] for line in r.stdout.splitlines()]

    return run


@pytest.mark.parametrize("which", [(), (0,), (3,), (4,), (5,), (0, 4), (4, 5), (1, 2, 5), (0, 1, 2, 3, 4, 5)], ids=str)
def test_every_word_is_cleared_by_one_call(call, which):
    timeout = 20  # TL_ERR_TIMEOUT
    assert call([7 + i if i in which else 0 for i in range(6)]) == [[timeout if which else 0] + [0] * 6, [0] * 7]


def test_a_failing_read_is_an_error_and_leaves_no_other_word(call):
    failed = 18  # TL_ERR_CUDA
    assert call([1, 0, 0, 0, 0, 1], failing=2) == [[failed] + [0] * 6] * 2
