"""What launchers settle once for each device, against a stand-in of the runtime's few calls with devices that differ."""
import shutil
import subprocess

import pytest

from sneppx_alg_b200 import _build

RUNTIME = r"""
#pragma once
#include <map>
#include <mutex>
#include <utility>
enum cudaError_t { cudaSuccess = 0, cudaErrorInvalidValue = 1 };
enum cudaFuncAttribute { cudaFuncAttributeMaxDynamicSharedMemorySize = 8 };
enum cudaDeviceAttr { cudaDevAttrMultiProcessorCount = 16 };
inline thread_local int now = 0;
inline std::mutex guard;
inline std::map<std::pair<int, const void*>, int> allowed;      // device and kernel -> bytes
inline int calls = 0, limit = 232448;
inline cudaError_t cudaGetDevice(int* d) { *d = now; return now < 0 ? cudaErrorInvalidValue : cudaSuccess; }
template <typename K>
cudaError_t cudaFuncSetAttribute(K k, cudaFuncAttribute, int bytes) {
  std::lock_guard<std::mutex> l(guard);
  ++calls;
  if (bytes > limit) return cudaErrorInvalidValue;
  allowed[{now, (const void*)k}] = bytes;
  return cudaSuccess;
}
inline cudaError_t cudaDeviceGetAttribute(int* v, cudaDeviceAttr, int dev) { *v = 100 + dev; return dev < 60 ? cudaSuccess : cudaErrorInvalidValue; }
"""

PROGRAM = r"""
#include <thread>
#include <vector>
#include <cstdio>
#include <cstdlib>
#include "per_device.h"
#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); std::exit(1); } } while (0)
static void first() {}
static void second() {}
int main() {
  using namespace sx;
  auto has = [](int dev, void (*k)()) { std::lock_guard<std::mutex> l(guard); return allowed[{dev, (const void*)k}]; };
  static SharedMemory smem;
  for (int dev : {0, 1, 0, 1, 63}) {
    now = dev;
    CHECK(smem.allow(1000, first, second) == 0 && has(dev, first) == 1000 && has(dev, second) == 1000);
  }
  CHECK(calls == 6);                                             // two kernels on three devices, once each
  now = 1;
  CHECK(smem.allow(2000, first, second) == 0 && has(1, first) == 2000 && has(0, first) == 1000);
  CHECK(smem.allow(1500, first, second) == 0 && has(1, first) == 2000 && calls == 8);      // a smaller size takes nothing back
  CHECK(smem.allow(limit + 1, first) == -10 && smem.allow(limit, first) == 0);             // a refusal is not kept
  for (int bad : {-1, 64}) {
    now = bad;
    CHECK(smem.allow(10, first) == -10);
  }
  static PerDevice number;
  int asked = 0;
  for (int dev : {2, 3, 2, 3}) {
    now = dev;
    CHECK(number.get([&](int d) { ++asked; return 10 * d; }) == 10 * dev);
  }
  CHECK(asked == 2);
  now = 4;
  CHECK(number.get([](int) { return -7; }) == -7 && number.get([](int) { return 5; }) == 5 && number.get([](int) { return 6; }) == 5);
  now = 1;
  CHECK(multiprocessors() == 101);
  now = 0;
  CHECK(multiprocessors() == 100);
  now = 61;
  CHECK(multiprocessors() == 148);
  // many threads, sizes that grow and shrink: what a thread was allowed stays allowed
  static SharedMemory shared;
  std::vector<std::thread> t;
  for (int i = 0; i < 8; ++i)
    t.emplace_back([&, i] {
      for (int k = 0; k < 2000; ++k) {
        now = 10 + k % 3;
        const int bytes = 100 + (k * 37 + i * 911) % 5000;
        if (shared.allow(bytes, first) || has(now, first) < bytes) std::exit(2);
      }
    });
  for (auto& x : t) x.join();
  std::puts("settled");
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs a C++ compiler")
def test_each_device_is_set_up_by_itself(tmp_path):
    (tmp_path / "cuda_runtime.h").write_text(RUNTIME)
    (tmp_path / "main.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-I", str(tmp_path), "-I", str(_build.CSRC), str(tmp_path / "main.cpp"), "-o", str(tmp_path / "main")],
                   check=True, timeout=120)
    r = subprocess.run([str(tmp_path / "main")], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "settled" in r.stdout, (r.returncode, r.stdout)
