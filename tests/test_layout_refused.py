"""What a step's layout makes of requests that cannot be right, by the planner's own function on the host: none of their numbers is left, so that nothing of
a refused request indexes the page tables."""
import shutil
import subprocess

import pytest

from spite_b200.kernels import build

MAIN = r"""
#include "drafts.cu"
#include <cstdio>
int main() {
    // rows of a table of four pages, pages of 16: what a row holds, its length, what it brings
    int held[] = {4, 5, 1 << 30, -1, 4, 4, 4, 2}, lengths[] = {50, 70, 0, 3, -1, -2147483647 - 1, 65, 20};
    int slots[] = {0, 1, 2, 3, 4, 5, 6, 7, 8, -2, 0, 1, 0}, fresh[] = {-1, -1, -1, -1, 1, 1, 1, 30, 1, 1, -2, 3, 2147483647}, stack[64], height = 0;
    LayoutParams p = {};
    p.held = held; p.lengths = lengths; p.slots = slots; p.new_tokens = fresh; p.free_pages = stack; p.n_free = &height;
    p.n_rows = 8; p.table_width = p.out_width = 4; p.n_pages = 64; p.n_requests = 13; p.n_tokens = 100; p.page_size = 16; p.window_kind = 2; p.window_size = 20;
    for (int s = 0; s < 13; ++s) {
        bool ok = false;
        const Request r = request_of(p, s, ok);
        printf("%d %d %d %d %d %d %d\n", ok, r.row, r.fresh, r.held, r.need, r.goes_to, r.goes);
    }
}
"""


@pytest.mark.skipif(shutil.which("g++") is None or not build._nvcc(), reason="needs the CUDA toolkit")
def test_nothing_is_left_of_a_refused_request(tmp_path):
    source = tmp_path / "plan.cu"
    source.write_text(MAIN)
    subprocess.run([build._nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-I", str(build.CSRC), "-o", str(tmp_path / "plan"), str(source)], check=True)
    out = subprocess.run([str(tmp_path / "plan")], check=True, capture_output=True, text=True).stdout
    got = [[int(v) for v in line.split()] for line in out.splitlines()]
    assert got[0] == [1, 0, -1, 4, 0, 4, 0]                   # ended: all of its pages go back
    refused = [0, -1, 0, 0, 0, 0, 0]
    assert got[1:7] == [refused] * 6                          # more pages than a row has (ended), a number below zero, longer than its pages
    assert got[7] == [1, 7, 30, 2, 4, 0, 0]                   # grows to four pages
    assert got[8:] == [refused] * 5
