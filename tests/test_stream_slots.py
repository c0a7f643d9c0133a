"""CPU test of the table that gives each stream a slot of its own (csrc/host.cuh), compiled with the host compiler."""
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
CUDA = Path("/usr/local/cuda/include")

CODE = r"""
#include <cassert>
#include <set>
#include <thread>
#include <vector>
#include "kernelfuser_b200/csrc/host.cuh"

static kf::host::StreamSlots<64> slots, shared_slots;

int main() {
    // two streams never share a slot, whatever their numbers, and each keeps its own however many calls lie between
    std::set<int> seen;
    std::vector<int> first;
    for (int i = 0; i < 64; ++i) {
        const int s = slots.of(1 + i % 3, 7 + 1024ull * (i / 3));
        assert(s >= 0 && s < 64 && seen.insert(s).second);
        first.push_back(s);
    }
    for (int turn = 0; turn < 5000; ++turn)
        for (int i = turn % 7; i < 64; i += 7) assert(slots.of(1 + i % 3, 7 + 1024ull * (i / 3)) == first[i]);
    // no slot is left for one more stream, and the others still have theirs
    for (int i = 0; i < 100; ++i) assert(slots.of(9, 5 + i) == -1);
    assert(slots.of(1, 7) == first[0]);
    // threads that meet
    std::vector<std::vector<int>> got(8, std::vector<int>(40));
    std::vector<std::thread> threads;
    for (int t = 0; t < 8; ++t)
        threads.emplace_back([&, t] {
            for (int turn = 0; turn < 200; ++turn)
                for (int i = 0; i < 40; ++i) got[t][i] = shared_slots.of(1, i);
        });
    for (auto& t : threads) t.join();
    for (int t = 1; t < 8; ++t) assert(got[t] == got[0]);
    assert(std::set<int>(got[0].begin(), got[0].end()).size() == 40);
}
"""


@pytest.mark.skipif(not shutil.which("g++") or not CUDA.exists(), reason="needs g++ and CUDA's headers")
def test_every_stream_has_a_slot_of_its_own(tmp_path):
    (tmp_path / "slots.cpp").write_text(CODE)
    exe = tmp_path / "slots"
    lib = CUDA.parent / "lib64"
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{ROOT}", f"-I{CUDA}", str(tmp_path / "slots.cpp"), "-o", str(exe), f"-L{lib}",
                    "-lcudart_static", "-ldl", "-lrt", "-lpthread"], check=True)
    subprocess.run([str(exe)], check=True, timeout=60)
