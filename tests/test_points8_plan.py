"""Which form of a kernel a size takes, and the sizes that are refused: the rules of annembed_amd/csrc/points8_plan.h, compiled for the host."""
import pathlib
import shutil
import subprocess

import pytest

from tests.test_gpu_points8_forms import GRADIENTS
from tests.test_gpu_points8_sums import SHAPES

ROOT = pathlib.Path(__file__).resolve().parent.parent
F32, BF16, F16 = range(3)
PROGRAM = r"""
#include "points8_plan.h"
#include <cinttypes>
#include <cstdio>
#include <cstring>
using namespace ae;
int main() {
    char what[16];
    uint64_t a[8];
    while (scanf("%15s", what) == 1) {
        for (auto& v : a)
            if (scanf("%" SCNu64, &v) != 1) return 1;
        if (!strcmp(what, "blocks")) {   // n dim type look
            const BlocksPlan p = blocks_plan(a[0], a[1], (uint32_t)a[2], a[3] != 0);
            printf("%d %u %d\n", p.trips, p.grid, (int)write_looks(a[0], a[1]));
        } else if (!strcmp(what, "range")) {   // rows lddc points size
            printf("%u\n", grad_range((uint32_t)a[0], (uint32_t)(a[1] * a[3]), (uint32_t)a[2], (uint32_t)a[3]));
        } else if (!strcmp(what, "product")) {   // m n dim: whether rows are few, points a workgroup takes then, the tile otherwise, tiles
            const ProductPlan p = product_plan(a[0], a[1], a[2]);
            printf("%d %d %d %llu\n", (int)few_rows(a[0], a[1], a[2]), (int)few_points(a[1], a[2]), p.tile, (unsigned long long)(p.tiles_m * p.tiles_n));
        } else if (!strcmp(what, "gradient")) {   // m n dim type
            const GradPlan p = grad_plan(a[0], a[1], a[2], (uint32_t)a[3]);
            printf("%u %llu %llu %u %llu\n", p.fr * 64, (unsigned long long)p.slices, (unsigned long long)p.per_slice, p.slices > 1 ? join_groups(p.slices) : 0, (unsigned long long)p.bytes);
        } else return 2;
    }
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no g++")
    at = tmp_path_factory.mktemp("plan")
    (at / "plan.cpp").write_text(PROGRAM)
    subprocess.run([cxx, "-std=c++17", "-Wall", "-Werror", "-O1", "-I", str(ROOT / "annembed_amd" / "csrc"), "-o", str(at / "plan"), str(at / "plan.cpp")], check=True)

    def ask(what, *numbers):
        line = " ".join([what] + [str(int(v)) for v in numbers] + ["0"] * (8 - len(numbers)))
        out = subprocess.run([str(at / "plan")], input=line + "\n", capture_output=True, text=True, check=True).stdout
        return tuple(int(v) if v.lstrip("-").isdigit() else float(v) for v in out.split())
    return ask


def test_launches_of_2_to_the_32_threads_are_refused(plan):
    """a workgroup of 256 threads takes 64 blocks of 16-bit rows, and of f32 beyond 2^27: 2^30 - 64 blocks are the most"""
    for kind in (F32, BF16, F16):
        assert plan("blocks", (1 << 30) - 64, 128, kind, 0)[:2] == (4, (1 << 24) - 1)
        for n, dim in (((1 << 30) - 63, 1), (1 << 30, 128), ((1 << 29) - 31, 129), ((1 << 31) - 1, 5), (1 << 20, 1 << 20)):
            assert plan("blocks", n, dim, kind, 0)[1] == 0
    assert plan("blocks", 1, 1, F32, 0)[:2] == (1, 1) and plan("blocks", 17, 128, BF16, 0)[:2] == (1, 2)


def test_blocks_a_group_of_lanes_takes(plan):
    assert plan("blocks", (1 << 20) - 5, 16, BF16, 0)[0] == 1 and plan("blocks", (1 << 20) + 77, 16, F16, 0)[0] == 4
    assert plan("blocks", (1 << 19) + 5, 130, BF16, 0)[0] == 4 and plan("blocks", 150001, 1000, BF16, 0)[0] == 4 and plan("blocks", 150001, 1000, F32, 0)[0] == 1
    assert plan("blocks", 4001, 1000, BF16, 1) == (1, 2001, 1) and plan("blocks", 5000, 4096, BF16, 1)[0] == 4
    for n, dim, looks in ((4096, 128, 1), (4097, 128, 0), (6000, 129, 1), (6001, 129, 0)):
        assert plan("blocks", n, dim, BF16, 0)[2] == looks


def test_the_gradient_reads_nothing_behind_its_tensor(plan):
    """a tile's buffer ends with its last row's last value, whether that is a whole dword or the first half of one"""
    for rows, lddc, points, size in ((1, 1, 1, 2), (1, 129, 129, 2), (64, 129, 129, 2), (128, 60001, 60001, 2), (5, 140, 129, 2), (64, 7, 7, 4), (3, 64, 64, 2)):
        assert plan("range", rows, lddc, points, size)[0] == ((rows - 1) * lddc + points) * size


def test_the_products_that_are_tested_take_every_form(plan):
    """few rows in 1, 2 and 4 tiles of 16, groups of points whole and shared; 64 x 64, 128 x 128 and 256 x 256 tiles"""
    forms = set()
    for m, n, dim in SHAPES:
        few, points, tile, _ = plan("product", m, n, dim)
        forms.add(("few", 1 if m <= 16 else 2 if m <= 32 else 4, points) if few else tile)
        forms.add(tile)   # (of another store's points: never few)
    assert forms == {("few", 1, 64), ("few", 1, 16), ("few", 2, 64), ("few", 2, 16), ("few", 4, 64), 64, 128, 256}


def test_the_borders_of_the_products_forms(plan):
    assert plan("product", 64 * 16, 64 * 24, 100)[2:] == (64, 384) and plan("product", 64 * 16, 64 * 24 + 1, 100)[2] == 128
    for m, n, dim, tile in ((4096, 4096, 897, 256), (4096, 4096, 896, 128), (4096, 3584, 2000, 256), (4096, 3328, 2000, 128), (4097, 4096, 2000, 128), (8192, 8192, 1024, 256),
                            (8192, 7936, 1024, 256), (300, 256 * 600, 2000, 128)):
        assert plan("product", m, n, dim)[2] == tile
    assert plan("product", 16, 32768, 784)[0] == 1 and plan("product", 65, 100, 28)[0] == 0 and plan("product", 64, 16384, 28)[0] == 1 and plan("product", 64, 16385, 28)[0] == 0
    for n in (1 << 30, (1 << 32) - 2):
        assert plan("product", 1, n, 1)[0] == 0


def test_the_gradients_that_are_tested_take_every_form(plan):
    forms, joins = set(), set()
    for m, n, dim in GRADIENTS:
        for kind in (F32, BF16, F16):
            rows, slices, per, groups, _ = plan("gradient", m, n, dim, kind)
            assert (slices - 1) * per < n <= slices * per and per % 64 == 0
            forms.add((kind, rows, slices > 1))
            joins.add(groups)
    assert forms == {(kind, rows, more) for kind in (F32, BF16, F16) for rows in (64, 128) for more in (False, True)} - {(F32, 128, False), (F32, 128, True)}
    assert joins == {0, 1, 4, 16, 64}


def test_scratch_of_the_gradient(plan):
    """the sums of all slices, rows of whole 16 bytes; none where one slice writes the result itself"""
    for m, n, dim in GRADIENTS + [(1, 1, 1), (1 << 20, 70, 3), (3, 1 << 26, 1 << 20)]:
        for kind in (F32, BF16, F16):
            rows, slices, per, _, size = plan("gradient", m, n, dim, kind)
            assert size == (slices * m * (-(-dim // 4) * 4) * 4 if slices > 1 else 0)
            assert per * (-(-dim // 16) * 16) <= 0x3FFF0000   # a slice's codes: 32-bit offsets reach them


def test_the_product_of_rows_far_apart_takes_tiles_of_128(plan):
    assert plan("product", 130, 8333, 200)[0] == 0 and plan("product", 130, 8333, 200)[2] == 128
