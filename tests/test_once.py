"""Per-device set-up of the launchers under several threads (CPU: once.cuh and the launchers' own state under the thread
sanitizer)."""

import re
import shutil
import subprocess

import pytest

from conftest import PKG_DIR

PROGRAM = """
#include <cstdio>
#include <thread>
#include <vector>
#include "once.cuh"
static std::atomic<int> sets{0};
static bool call(int device) {
  static tl::Once<4> ready;
  return ready(device, [] { return ++sets > 0; });
}
int main() {
  tl::Once<2> once;
  bool ok = !once(0, [] { return false; }) && once(0, [] { return true; }) && once(0, [] { return false; }) &&
            !once(1, [] { return false; }) && !once(-1, [] { return true; }) && !once(2, [] { return true; });
  std::vector<std::thread> threads;
  std::atomic<int> failed{0};
  for (int t = 0; t < 8; ++t)
    threads.emplace_back([&] {
      for (int i = 0; i < 1000; ++i)
        for (int d = 0; d < 4; ++d) failed += !call(d);
    });
  for (auto& t : threads) t.join();
  ok = ok && !failed && sets >= 4 && sets <= 32;
  puts(ok ? "fine" : "wrong");
}
"""


def test_threads_that_come_first_together(tmp_path):
    if not shutil.which("g++"):
        pytest.skip("no g++")
    (tmp_path / "once.cc").write_text(PROGRAM)
    built = subprocess.run(["g++", "-std=c++17", "-g", "-O1", "-fsanitize=thread", "-I", str(PKG_DIR / "csrc"),
                            str(tmp_path / "once.cc"), "-o", str(tmp_path / "once")], capture_output=True, text=True)
    if "tsan" in built.stderr and "cannot find" in built.stderr:
        pytest.skip("no thread sanitizer")
    assert built.returncode == 0, built.stderr
    r = subprocess.run([str(tmp_path / "once")], capture_output=True, text=True)
    if "unexpected memory mapping" in r.stderr:
        pytest.skip("the thread sanitizer cannot run here")
    assert r.returncode == 0 and r.stdout.strip() == "fine", r.stderr


@pytest.mark.parametrize("source", ["paged.cu", "paged_attn.cu", "logprobs.cu", "serving.cuh"])
def test_the_serving_launchers_keep_no_plain_state(source):
    """A static of a host function is constant, atomic or a Once."""
    text = re.sub(r"//.*", "", (PKG_DIR / "csrc" / source).read_text())
    plain = [m for m in re.findall(r"^\s+static (?!constexpr|const |_?assert)[^;(]*;", text, flags=re.M)
             if "Once<" not in m and "std::atomic<" not in m]
    assert not plain
