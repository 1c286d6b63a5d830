"""The K tiles that the fp8 x fp8 kernels for few rows load, and the scales they read, stay inside the operands: their walk
(csrc/wq_f8f8_walk.h), compiled for the host and stepped as the kernels step it."""
import os
import subprocess

import pytest

from composable_kernel_amd import capi

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "composable_kernel_amd", "csrc")

DRIVER = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "wq_f8f8_walk.h"

// K, k per slice, slices, waves of a workgroup, tiles in flight, workgroups
int main(int, char** v)
{
    const int K = std::atoi(v[1]), per = std::atoi(v[2]), slices = std::atoi(v[3]), waves = std::atoi(v[4]), depth = std::atoi(v[5]), groups = std::atoi(v[6]);
    const int kblocks = (K + 127) / 128;
    for(int z = 0; z < slices; ++z)
        for(int block = 0; block < groups; ++block)
        {
            const int k0 = z * per, k1 = k0 + per < K ? k0 + per : K, ntiles = (k1 - k0 + 127) >> 7;
            const wq::F8F8Walk walk(ntiles, block * 11u);
            if(walk.empty())
                continue;
            std::vector<int> seen(ntiles, 0);
            for(int wave = 0; wave < waves; ++wave)
            {
                const int mine = ntiles > wave ? (ntiles - wave + waves - 1) / waves : 0;
                for(int j = 0; j < mine + depth; ++j)
                {
                    const int step = wave + j * waves, column = k0 / 128 + walk.scales(step);
                    if(column < k0 / 128 || column >= kblocks || column * 128 >= k1)
                        return std::printf("slice %d reads scale %d of %d\n", z, column, kblocks), 1;
                    if(j < mine && (walk.tile(step) < 0 || walk.tile(step) >= ntiles || walk.scales(step) != walk.tile(step) || seen[walk.tile(step)]++))
                        return std::printf("slice %d step %d takes tile %d of %d\n", z, step, walk.tile(step), ntiles), 1;
                }
            }
            for(int n : seen)
                if(n != 1)
                    return std::printf("slice %d leaves a tile out\n", z), 1;
        }
    return 0;
}
"""


@pytest.fixture(scope="module")
def driver(tmp_path_factory):
    d = tmp_path_factory.mktemp("walk")
    (d / "walk.cpp").write_text(DRIVER)
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-I", CSRC, "-o", str(d / "walk"), str(d / "walk.cpp")])
    return str(d / "walk")


@pytest.mark.parametrize("k,k_batch", [(128, 1), (16, 3), (128, 65535), (256, 3), (256, 8), (256, 1000), (384, 2), (1040, 5), (2048, 32), (4096, 3), (4112, 33), (8192, 7)])
@pytest.mark.parametrize("waves,depth", [(4, 2), (8, 1), (8, 2), (16, 1)])
def test_every_tile_once_and_no_scale_outside_the_table(driver, k, k_batch, waves, depth):
    r = subprocess.run([driver, *map(str, (k, capi.splitk_kread(k, k_batch, 128), k_batch, waves, depth, 40))], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout


def test_slices_behind_the_end_are_accepted():
    p = capi.f8_problem(0x10000, 0x10000, 0x10000, 0x10000, 0x10000, 16, 512, 256, k_batch=8)
    assert capi.kernel_name(p).startswith("wq_gemm_f8f8_skinny") and "KBatch8" in capi.type_string(p)
