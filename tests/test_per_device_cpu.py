"""What the kernels keep per device (csrc/per_device.h): only what was found
without an error, each device for itself, and once among threads."""
import subprocess
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "cottus-runtime_b200" / "csrc"

PROGRAM = r"""
#include <cassert>
#include <cstdio>
#include <thread>
#include <vector>
#include "per_device.h"
enum Err { kOk = 0, kBusy = 1, kRange = 2 };
static cb200::PerDevice<int, Err, 4> table;
int main() {
    int v = -1, calls = 0;
    auto fails = [&](int& x) { ++calls; x = 99; return kBusy; };
    auto finds = [&](int& x) { ++calls; x = 7; return kOk; };
    assert(table.get(1, v, kRange, fails) == kBusy && v == -1 && calls == 1);   // reported,
    assert(table.get(1, v, kRange, fails) == kBusy && calls == 2);              // not kept,
    assert(table.get(1, v, kRange, finds) == kOk && v == 7 && calls == 3);      // and forgotten
    assert(table.get(1, v, kRange, fails) == kOk && v == 7 && calls == 3);      // what was found stays
    assert(table.get(0, v, kRange, fails) == kBusy && calls == 4);              // of its own device only
    assert(table.get(4, v, kRange, finds) == kRange && table.get(-1, v, kRange, finds) == kRange && calls == 4);
    std::atomic<int> found{0};
    std::vector<std::thread> threads;
    for (int i = 0; i < 8; ++i)
        threads.emplace_back([&] {
            int x = 0;
            assert(table.get(2, x, kRange, [&](int& y) { ++found; y = 5; return kOk; }) == kOk && x == 5);
        });
    for (auto& t : threads) t.join();
    assert(found == 1);
    std::puts("ok");
}
"""


def test_failures_are_not_kept(tmp_path):
    src, exe = tmp_path / "per_device.cpp", tmp_path / "per_device"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-I", str(CSRC), str(src), "-o", str(exe)], check=True)
    assert subprocess.run([str(exe)], capture_output=True, text=True, timeout=60).stdout == "ok\n"
