"""The "done once per device" flags of the launch code (whisperjav_amd/csrc/attr_once.hpp), compiled for the host with a stand-in for hipGetDevice."""
import os
import shutil
import subprocess

import pytest

from whisperjav_amd import build

CXX = shutil.which("g++") or shutil.which("clang++")
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")
pytestmark = pytest.mark.skipif(CXX is None or not os.path.exists(os.path.join(ROCM, "include", "hip", "hip_runtime_api.h")), reason="no host compiler or no HIP headers")

PROGRAM = """
#include <hip/hip_runtime_api.h>
#include <stdio.h>
#include <thread>
#include <vector>
static thread_local int current = 0;
static inline hipError_t stand_in(int* d) { *d = current; return hipSuccess; }
#define hipGetDevice stand_in
#include "%s"
int main() {
  wj::AttrOnce flag;
  auto on = [](int d) { current = d; };
  // two threads' turns: device 0 asks, device 1 asks, device 0 is done
  on(0); if (!flag.need()) return 1;
  on(1); if (!flag.need()) return 2;
  on(0); flag.done();
  if (flag.need()) return 3;
  on(1); if (!flag.need()) return 4;            // device 1 has not set its attribute yet
  flag.done();
  if (flag.need()) return 5;
  on(2); if (!flag.need()) return 6;
  // and threads that run at once: none is told that its device is done before it said so itself
  for (int round = 0; round < 200; ++round) {
    wj::AttrOnce f;
    int wrong = 0;
    std::vector<std::thread> all;
    std::vector<int> bad(8, 0);
    for (int d = 0; d < 8; ++d) all.emplace_back([&, d] { on(d); bad[d] = !f.need(); f.done(); bad[d] += f.need(); });
    for (auto& t : all) t.join();
    for (int b : bad) wrong += b;
    if (wrong) return 7;
  }
  return 0;
}
"""


def test_each_device_answers_for_itself(tmp_path):
    (tmp_path / "once.cpp").write_text(PROGRAM % (build.CSRC / "attr_once.hpp"))
    subprocess.run([CXX, "-std=c++17", "-O1", "-D__HIP_PLATFORM_AMD__", "-I", os.path.join(ROCM, "include"), str(tmp_path / "once.cpp"), "-o", str(tmp_path / "once"),
                    "-pthread"], check=True)
    assert subprocess.run([str(tmp_path / "once")]).returncode == 0
