"""The plan of block-scaled e4m3 products (csrc/f8blk_plan.cuh, compiled here for the host) over shapes of every size and three tables of resident
clusters: what the kernels have room for, no split whose clusters cannot all be resident, no part of K under two blocks, and estimates that
stay numbers at the largest sizes."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "paddock_b200", "csrc")
SRC = r"""
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <initializer_list>
#include "f8blk_plan.cuh"
using namespace f8blk;
static void fail(const char* what, int planes, unsigned k, unsigned n, unsigned m, const Plan& p) {
    std::printf("%s: planes %d K %u N %u tokens %u: kernel %u cols %u split %u\n", what, planes, k, n, m, p.kernel, p.cols, p.split);
    std::exit(1);
}
int main() {
    const uint32_t caps[3][9] = {{0, 148, 74, 48, 36, 28, 22, 18, 16}, {0, 148, 74, 45, 33, 26, 22, 15, 15}, {0, 16, 8, 0, 4, 0, 0, 0, 1}};
    unsigned long long plans = 0, reached = 0;
    for (const auto& cap : caps) {
        const uint32_t* const resident[2] = {cap, cap};
        const uint32_t sms = cap[1];
        for (int planes = 1; planes <= 2; ++planes)
            for (unsigned k : {16u, 128u, 144u, 400u, 1040u, 2880u, 5120u, 17408u, 262144u, 0x7fffff00u})
                for (unsigned n : {1u, 16u, 128u, 130u, 1024u, 2880u, 5003u, 17408u, 25600u, 262144u, 0x7fffff00u})
                    for (unsigned m : {1u, 7u, 31u, 32u, 33u, 48u, 64u, 65u, 200u, 600u, 2000u, 8192u, 1u << 20, 0x7fffff00u}) {
                        const Plan p = choose(planes, k, n, m, resident, 8u, sms);
                        ++plans;
                        const uint64_t blocks = (k + 127ull) / 128, tiles_n = (n + 127ull) / 128;
                        if (p.kernel == 1) {
                            if (p.cols != 32 && p.cols != 64) fail("tokens of a tile", planes, k, n, m, p);
                            if (p.cols == 64 && m <= 32) fail("half-empty tile", planes, k, n, m, p);
                            const uint64_t tiles = (m + (uint64_t)p.cols - 1) / p.cols * tiles_n;
                            if (p.split < 1 || p.split > 8 || (p.split > 1 && blocks < 2ull * p.split)) fail("part of K", planes, k, n, m, p);
                            if (p.split > 1 && tiles > 2ull * cap[p.split]) fail("clusters resident at once", planes, k, n, m, p);
                            const double us = split_us(planes, m < p.cols ? m : p.cols, tiles, (uint32_t)blocks, p.cols, p.split, sms);
                            if (!std::isfinite(us) || us <= 0) fail("estimate", planes, k, n, m, p);
                        } else {
                            if (p.kernel != 2 || p.split != 1) fail("kernel", planes, k, n, m, p);
                            if (p.cols != 256 && !(p.cols == 128 && planes == 1)) fail("channels of a tile", planes, k, n, m, p);
                            const double us = wide_us(planes, (m + 127ull) / 128 * tiles_n, (uint32_t)blocks, p.cols, sms);
                            if (!std::isfinite(us) || us <= 0) fail("estimate", planes, k, n, m, p);
                        }
                        reached |= 1ull << ((planes - 1) * 8 + (p.kernel - 1) * 4 + (p.cols == 64 || p.cols == 256) * 2 + (p.split > 1));
                    }
    }
    // one plane: both tiles of both kernels, with and without a split; gated: the same without wide tiles of 128
    for (int bit : {0, 1, 2, 3, 4, 6, 8, 9, 10, 11, 14})
        if (!(reached >> bit & 1)) { std::printf("no shape takes plan %d\n", bit); return 1; }
    std::printf("%llu plans\n", plans);
}
"""


def test_plans_of_every_size(tmp_path):
    src, exe = tmp_path / "plan.cc", tmp_path / "plan"
    src.write_text(SRC)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout + run.stderr
    assert int(run.stdout.split()[0]) == 3 * 2 * 10 * 11 * 14
