"""Work of any length is cut into launches that a grid can hold, each piece once and in order (CPU only: the header is
compiled by itself, with limits small enough to be met)."""
import os
import subprocess

from conftest import ROOT

CSRC = os.path.join(ROOT, "comfyui-weightferry_amd", "csrc")
PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "grids.h"
#define CHECK(c) do { if (!(c)) { std::printf("line %d: %s\n", __LINE__, #c); return 1; } } while (0)

int main() {
    CHECK(wf::kGridMost * 256 < (1LL << 32));
    for (int64_t most : {1LL, 7LL, 1000LL, (long long)wf::kGridMost})
        for (int64_t wgs : {0LL, 1LL, 6LL, 7LL, 8LL, 21LL, 1LL << 26, (1LL << 26) + 5}) {
            if (wgs / most > 100000) continue;
            int64_t at = 0;
            wf::over_grids(wgs, most, [&](int64_t first, uint32_t n) {
                if (first != at || n == 0 || n > most) std::exit(2);
                at += n;
            });
            CHECK(at == wgs);
        }
    std::srand(1);
    for (int round = 0; round < 3000; round++) {
        const int block = 1 + std::rand() % 5, wg_blocks = 1 + std::rand() % 4, tensors = 1 + std::rand() % 6;
        const int64_t most = 1 + std::rand() % 12;
        std::vector<int64_t> sizes(std::rand() % 20);
        for (auto& n : sizes) n = std::rand() % 3 ? std::rand() % 40 : std::rand() % 600;
        std::vector<int64_t> done(sizes.size());
        int used = 0;
        int64_t next = 0;
        size_t last = 0;
        bool ok = true;
        wf::over_tensors((int64_t)sizes.size(), block, wg_blocks, tensors, most, [&](int64_t i) { return sizes[i]; },
            [&](int slot, int64_t i, int64_t first, int64_t n, uint32_t wg) {
                ok = ok && slot == used && wg == next && first == done[i] && n > 0 && (size_t)i >= last &&
                     first % wg_blocks == 0;
                last = i, used++, done[i] += n, next += (n + wg_blocks - 1) / wg_blocks;
            },
            [&](int parts, uint32_t wgs) {
                ok = ok && parts == used && parts > 0 && parts <= tensors && wgs == next && wgs <= most;
                used = 0, next = 0;
            });
        CHECK(ok && used == 0);
        for (size_t i = 0; i < sizes.size(); i++) CHECK(done[i] == (sizes[i] + block - 1) / block);
    }
    // a tensor past one grid at the real limits
    int64_t blocks = 0;
    int launches = 0;
    wf::over_tensors(2, 256, 8, 96, wf::kGridMost, [](int64_t) { return (1LL << 36) + 1; },
        [&](int, int64_t, int64_t, int64_t n, uint32_t) { blocks += n; },
        [&](int, uint32_t wgs) { launches++; if (wgs > wf::kGridMost) std::exit(3); });
    CHECK(blocks == 2 * ((1LL << 28) + 1) && launches == 5);
    std::puts("ok");
    return 0;
}
"""


def test_launches_cover_the_work(tmp_path):
    src, exe = tmp_path / "grids.cpp", tmp_path / "grids"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert (out.returncode, out.stdout.strip()) == (0, "ok"), out.stdout
