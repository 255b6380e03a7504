"""CPU test of the linear kernels' tile arithmetic (csrc/bcjr_tiles.cuh), which
is compiled for the host here with traps on signed overflow."""
import subprocess

from quant_2bit_b200.build import CSRC

PROGRAM = r"""
#include "bcjr_tiles.cuh"
#include <cstdio>
#include <cstdlib>

using namespace bcjr::mm;

static void need(bool ok, const char *what, long rows, long c) {
    if (!ok) {
        std::printf("%s: rows %ld tile %ld\n", what, rows, c);
        std::exit(1);
    }
}

// The tiles of one group as the kernels walk them: each has 1 to COLS rows, the
// next one starts where it ends, and they end with the group.
template <int COLS>
static void check(int rows, int step) {
    const int tiles = col_tiles<COLS>(rows), share = tile_share(rows, tiles, step);
    need(tiles >= 1 && share >= 1 && share <= COLS && share % step == 0, "share", rows, share);
    for (int c = 0; c < tiles; c = (tiles > 4000 && c == 1000) ? tiles - 1000 : c + 1) {
        const int col0 = c * share, left = rows - col0, valid = share < left ? share : left;
        need(valid >= 1 && valid <= COLS, "valid", rows, c);
        need(c < tiles - 1 ? valid == share : col0 + valid == rows, "end", rows, c);
        const int ncols = (valid + step - 1) & ~(step - 1);
        need(ncols >= step && ncols <= COLS, "ncols", rows, c);
    }
    need(max_col_tiles<COLS>(rows, 1) == tiles, "most", rows, 1);
    need(max_col_tiles<COLS>(rows, 2) >= tiles, "most", rows, 2);
}

int main() {
    const int last = int(kMaxRows);
    const int more[] = {1 << 24, (1 << 30) + 1, 2100000000, 2114445437, 2114445438, 2139127679, 2139127680,
                        2139127681, last - 257, last - 255, last - 33, last - 31, last - 1, last};
    for (int step = 16; step <= 32; step *= 2) {
        for (int rows = 1; rows <= 5000; ++rows) {
            check<64>(rows, step);
            check<128>(rows, step);
            check<256>(rows, step);
        }
        for (int rows : more) {
            check<64>(rows, step);
            check<128>(rows, step);
            check<256>(rows, step);
        }
    }
    std::puts("ok");
}
"""


def test_tiles_cover_a_group_of_any_size(tmp_path):
    source, program = tmp_path / "tiles.cpp", tmp_path / "tiles"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fsanitize-undefined-trap-on-error",
                    "-x", "c++", "-I", CSRC, str(source), "-o", str(program)], check=True)
    run = subprocess.run([str(program)], capture_output=True, text=True)
    assert run.returncode == 0 and run.stdout.strip() == "ok", (run.returncode, run.stdout)


def test_the_kernels_use_this_arithmetic():
    """No other copy of it, and the entry points accept no more rows."""
    import os
    text = {n: open(os.path.join(CSRC, n)).read() for n in ("bcjr_mm.cuh", "bcjr_fp8.cu", "bcjr_grouped.cu")}
    assert "tile_share(" in text["bcjr_mm.cuh"] and "rows + ct - 1" not in text["bcjr_mm.cuh"]
    assert all("kMaxRows" in text[n] and "0x7fffff00" not in text[n] for n in ("bcjr_fp8.cu", "bcjr_grouped.cu"))
