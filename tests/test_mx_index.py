"""Index arithmetic of the microscaled kernels at the ends of what their calls accept, on the CPU:
the kernels' own functions (csrc/mx.cuh), compiled into a small host program."""
import os
import subprocess

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
pytestmark = pytest.mark.skipif(not os.path.exists(NVCC), reason="no nvcc")


def run(tmp_path, body):
    """What `body`, the inside of main(), prints."""
    src, exe = tmp_path / "index.cu", tmp_path / "index"
    src.write_text("#include <cstdio>\n#include \"mx.cuh\"\nusing namespace opure;\nint main() {\n" + body + "\n}\n")
    subprocess.run([NVCC, "-std=c++17", "-O1", "--expt-relaxed-constexpr", "-gencode", "arch=compute_100a,code=sm_100a",
                    f"-I{REPO}/include", f"-I{REPO}/opure-voxelengine_b200/csrc", "-o", str(exe), str(src)], check=True)
    return subprocess.run([str(exe)], check=True, capture_output=True, text=True, timeout=60).stdout.split()


def test_row_of_a_warp_does_not_wrap(tmp_path):
    """256 threads a block, 8 rows each: row 2^27 is the first whose threads' flat index needs more
    than 32 bits; 0x7fffffff rows are the most that the norm takes."""
    got = run(tmp_path, """
    for (uint32_t row : {0u, 9u, (1u << 27) - 1, 1u << 27, (1u << 27) + 13, 0x7ffffffeu})
        for (uint32_t lane : {0u, 31u}) printf("%u ", mx_warp_row(row / 8, row % 8 * 32 + lane, 256) - row);""")
    assert got == ["0"] * 12


def test_norm_columns_do_not_wrap(tmp_path):
    """The norm's two loops over a long row, counted as the kernel counts them, at the most columns
    that its call takes: as many passes as cover the row, no column twice. Longer rows, whose last
    step would pass 2^32 (the loop would not end), are refused."""
    got = run(tmp_path, """
    const uint32_t step = kMxNormStep, most = 0u - step;
    printf("%d%d%d%d ", mx_norm_takes(0x7fffffff, most), mx_norm_takes(1, most + 1), mx_norm_takes(1, 0xffffff80u), mx_norm_takes(0x80000000u, 1));
    for (uint32_t cols : {20000u, most - 130, most - 7, most})
        for (uint32_t c0 : {0u, 8u, step - 8}) {
            const uint32_t kp = mx_kp(cols);
            uint64_t first = 0, second = 0, limit = 600000;
            bool ok = true;
            for (uint32_t c = c0; c < cols && first < limit; c += step) ok &= c == c0 + step * first++;
            for (uint32_t b = 0; b < kp && second < limit; b += step) ok &= b + c0 == c0 + step * second++;
            printf("%d ", ok && first == (uint64_t(cols) - c0 + step - 1) / step && second == (uint64_t(kp) + step - 1) / step);
        }""")
    assert got == ["1000"] + ["1"] * 12
