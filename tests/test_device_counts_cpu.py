"""Counts that are asked of a device once (csrc/device_counts.h) and what the acceptance's launch form is chosen by: no caller sees one that is still being asked
for, devices do not answer for one another, a failed query is not kept.  No GPU."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(__file__), "..", "glm53f-afd_b200", "csrc")

PROGRAM = r"""
#include "device_counts.h"
#include <chrono>
#include <cstdio>
#include <thread>
#include <vector>
#define CHECK(x) do { if (!(x)) { printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)
int main() {
    {   // many callers while the first query is under way
        static kda::DeviceCounts<2> counts;
        std::atomic<int> wrong{0};
        std::vector<std::thread> all;
        for (int i = 0; i < 16; ++i)
            all.emplace_back([&] {
                for (int j = 0; j < 50; ++j)
                    if (counts.get(0, 1, [] { std::this_thread::sleep_for(std::chrono::milliseconds(5)); return 9; }) != 9) ++wrong;
            });
        for (auto& t : all) t.join();
        CHECK(wrong == 0);
    }
    kda::DeviceCounts<2> counts;
    int asked = 0;
    auto answer = [&](int n) { return [&asked, n] { ++asked; return n; }; };
    CHECK(counts.get(0, 0, answer(4)) == 4 && counts.get(0, 0, answer(5)) == 4 && asked == 1);
    CHECK(counts.get(0, 1, answer(6)) == 6 && counts.get(1, 0, answer(7)) == 7 && counts.get(0, 0, answer(8)) == 4 && counts.get(1, 0, answer(8)) == 7 && asked == 3);
    CHECK(counts.get(2, 0, answer(-1)) == 0 && counts.get(2, 0, answer(3)) == 3 && counts.get(2, 0, answer(8)) == 3 && asked == 5);  // a failure is not kept
    CHECK(counts.get(3, 1, answer(0)) == 0 && counts.get(3, 1, answer(2)) == 0 && asked == 6);                                       // none is an answer
    CHECK(counts.get(-1, 0, answer(2)) == 2 && counts.get(500, 0, answer(3)) == 3 && counts.get(500, 0, answer(4)) == 4);            // no such place
    puts("counts as asked");
}
"""


def test_counts(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no g++")
    (tmp_path / "x.cpp").write_text(PROGRAM)
    subprocess.check_call([gxx, "-std=c++17", "-O1", "-Wall", "-Werror", "-I" + CSRC, "-pthread", "-o", str(tmp_path / "x"), str(tmp_path / "x.cpp")])
    r = subprocess.run([str(tmp_path / "x")], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "counts as asked" in r.stdout, r.stdout


def test_the_launch_form_is_chosen_by_it():
    with open(os.path.join(CSRC, "spec_accept.cu")) as f:
        fit = f.read().split("int fit() {", 1)[1].split("int run(", 1)[0]
    assert "DeviceCounts" in fit and "static int" not in fit and "cudaGetDevice" in fit
