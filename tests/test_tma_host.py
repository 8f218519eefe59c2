"""The host side of the TMA tensor maps, compiled alone with a driver query of the test's own."""

from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

from mednext_accel_b200 import _build

SOURCE = r"""
#include <chrono>
#include <cstdio>
#include <thread>
#include <vector>

#include "tma_host.h"

static std::atomic<int> queries{0};
static CUresult encode(...) { return CUDA_SUCCESS; }

// The runtime's query, slow: what a process's first calls from several threads meet.
extern "C" cudaError_t cudaGetDriverEntryPoint(const char*, void** p, unsigned long long,
                                               cudaDriverEntryPointQueryResult* q) {
  ++queries;
  std::this_thread::sleep_for(std::chrono::milliseconds(300));
  *p = reinterpret_cast<void*>(&encode);
  *q = cudaDriverEntryPointSuccess;
  return cudaSuccess;
}

int main() {
  std::atomic<int> without{0};
  std::vector<std::thread> threads;
  for (int i = 0; i < 8; ++i)
    threads.emplace_back([&] {
      if (mednext::tma::encode_fn() == nullptr) ++without;
    });
  for (auto& t : threads) t.join();
  std::printf("%d %d", queries.load(), without.load());
}
"""


def test_threads_whose_first_calls_meet_all_get_the_encoder(tmp_path):
    compiler, nvcc = shutil.which("g++"), Path(_build.nvcc())
    if compiler is None:
        pytest.skip("needs g++")
    (tmp_path / "main.cpp").write_text("#include <atomic>\n" + SOURCE)
    program = tmp_path / "main"
    subprocess.run([compiler, "-std=c++17", "-pthread", f"-I{_build.CSRC}", f"-I{nvcc.resolve().parents[1] / 'include'}",
                    str(tmp_path / "main.cpp"), "-o", str(program)], check=True)
    run = subprocess.run([str(program)], check=True, capture_output=True, text=True, timeout=60)
    assert run.stdout == "1 0"  # one query, no thread without
