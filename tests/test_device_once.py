"""CPU tier: what a launcher sets once on a device is set before any thread's launch (livecc_amd/csrc/device_once.h), compiled with the host compiler against a stand-in for the device."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "livecc_amd", "csrc")
PROGRAM = r"""
#include <chrono>
#include <cstdio>
#include <thread>
#include <vector>
thread_local int device = 0;
static int hipGetDevice(int* d) { *d = device; return 0; }
#include "device_once.h"

static lcc::DeviceOnce once;
static std::atomic<int> set[2], times[2], early{0};
static void launch(int d) {
  device = d;
  if (auto turn = once.first()) {
    times[d]++;
    std::this_thread::sleep_for(std::chrono::milliseconds(100));      // another thread comes meanwhile
    set[d] = 1;
  }
  if (!set[d]) early++;
}
int main() {
  std::vector<std::thread> all;
  for (int i = 0; i < 16; ++i) all.emplace_back(launch, i & 1);
  for (auto& t : all) t.join();
  for (int i = 0; i < 4; ++i) launch(i & 1);
  std::printf("%d %d %d\n", times[0].load(), times[1].load(), early.load());
  return 0;
}
"""


def test_no_thread_launches_before_the_attribute_is_set(tmp_path):
    cxx = shutil.which("g++") or shutil.which("c++") or shutil.which("clang++")
    if cxx is None:
        pytest.skip("no host C++ compiler")
    (tmp_path / "once.cpp").write_text(PROGRAM)
    subprocess.run([cxx, "-std=c++17", "-O1", "-pthread", "-I", CSRC, str(tmp_path / "once.cpp"), "-o", str(tmp_path / "once")], check=True, capture_output=True)
    out = subprocess.run([str(tmp_path / "once")], check=True, capture_output=True, text=True, timeout=60).stdout.split()
    assert out == ["1", "1", "0"], "set once on either device, no launch ahead of it"
