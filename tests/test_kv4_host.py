"""The 4-bit KV cache without a GPU: page sizes, the layout's offsets (csrc/kv4.cuh, compiled into a
small host program, against the tests' own), what a layout is refused for, and the tests' reference
against values worked out by hand."""
import os
import subprocess

import numpy as np
import pytest

import kv4_reference as ref
from voxelengine import cuda as cu

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")


def run(tmp_path, body):
    """What `body`, the inside of main(), prints."""
    src, exe = tmp_path / "kv4.cu", tmp_path / "kv4"
    src.write_text("#include <cstdio>\n#include \"kv4.cuh\"\nusing namespace opure;\nint main() {\n" + body + "\n}\n")
    subprocess.run([NVCC, "-std=c++17", "-O1", "--expt-relaxed-constexpr", "-gencode", "arch=compute_100a,code=sm_100a",
                    f"-I{REPO}/include", f"-I{REPO}/opure-voxelengine_b200/csrc", "-o", str(exe), str(src)], check=True)
    return subprocess.run([str(exe)], check=True, capture_output=True, text=True, timeout=60).stdout.split()


@pytest.mark.parametrize("n_kv,hd,page,want", [
    (1, 64, 16, 1152), (3, 64, 64, 3 * 4 * 1152), (8, 128, 128, 8 * 8 * 2304), (65535, 128, 128, 65535 * 8 * 2304),
    (0, 64, 64, 0), (1, 96, 64, 0), (1, 64, 48, 0), (65536, 64, 16, 0),
])
def test_page_bytes(n_kv, hd, page, want):
    assert cu.kv4_page_bytes(n_kv, hd, page) == want


def test_scratch_of_any_sizes():
    """No entry has more queries than there are rows; 0 for more work than a grid takes, at sizes that leave 32 bits
    (or whose tiles are a multiple of 2^32)."""
    size = cu.kv4_attention_scratch_bytes
    assert size(1, 8, 2 ** 32 - 1, 4, 2, 64, 5000) == size(1, 8, 8, 4, 2, 64, 5000) > 16
    assert size(1, 40, 2 ** 31, 512, 1, 64, 5000) == size(1, 40, 40, 512, 1, 64, 5000) > 16
    assert size(1, 2 ** 31, 2 ** 31, 512, 1, 64, 5000) == 0
    assert size(2 ** 32 - 1, 2 ** 31, 2 ** 20, 512, 64, 64, 5000) == 0
    assert size(2 ** 32 - 1, 2 ** 32 - 1, 1, 1, 1, 64, 5000) == 0
    assert size(2 ** 20, 2 ** 20, 1, 8, 8, 64, 5000, 256) == 16  # enough work without splits


@pytest.mark.parametrize("hd", [64, 128])
def test_offsets_cover_each_byte_once(hd):
    assert sorted(np.concatenate(ref.offsets(hd), 1).ravel()) == list(range(18 * hd))


@pytest.mark.skipif(not os.path.exists(NVCC), reason="no nvcc")
def test_kernel_offsets_are_the_layout(tmp_path):
    got = np.array(run(tmp_path, """
    for (uint32_t hd : {64u, 128u})
        for (uint32_t t = 0; t < 16; ++t) {
            for (uint32_t b = 0; b < hd / 16; ++b) for (uint32_t j = 0; j < 8; ++j) printf("%u ", kv4_key_at(t, b) + j);
            for (uint32_t o = 0; o < hd / 8; ++o) for (uint32_t j = 0; j < 4; ++j) printf("%u ", kv4_value_at(hd, t, o) + j);
            for (uint32_t b = 0; b < hd / 16; ++b) printf("%u ", kv4_key_scale_at(hd, t, b));
            for (uint32_t b = 0; b < hd / 16; ++b) printf("%u ", kv4_value_scale_at(hd, t, b));
        }"""), int)
    want = np.concatenate([np.concatenate(ref.offsets(hd), 1).ravel() for hd in (64, 128)])
    assert np.array_equal(got, want)


@pytest.mark.skipif(not os.path.exists(NVCC), reason="no nvcc")
def test_layout_checks(tmp_path):
    """Status of a layout (made of a pointer that is never followed) for each wrong field."""
    got = run(tmp_path, """
    auto make = [] {
        opure_kv4_layout l{};
        l.pool = reinterpret_cast<uint8_t *>(256);
        l.page_table = reinterpret_cast<const int32_t *>(256);
        l.n_pages = 4; l.max_pages = 4; l.page_size = 64; l.n_kv = 2; l.head_dim = 64;
        return l;
    };
    auto say = [&](auto change) { opure_kv4_layout l = make(); change(l); printf("%d ", int(kv4_check(l))); };
    say([](auto &) {});
    say([](auto &l) { l.k_scale = 0.25f; l.v_scale = 1024.f; l.ring = 4; l.head_dim = 128; l.page_size = 16; });
    say([](auto &l) { l.k_scale = 0x1p-60f; l.v_scale = 0x1p60f; });
    say([](auto &l) { l.pool = nullptr; });
    say([](auto &l) { l.pool += 8; });
    say([](auto &l) { l.page_table = nullptr; });
    say([](auto &l) { l.n_pages = 0; });
    say([](auto &l) { l.max_pages = 0; });
    say([](auto &l) { l.ring = 5; });
    say([](auto &l) { l.k_scale = 3.f; });
    say([](auto &l) { l.v_scale = -1.f; });
    say([](auto &l) { l.v_scale = 0x1p61f; });
    say([](auto &l) { l.k_scale = 0x1p-61f; });
    say([](auto &l) { l.k_scale = INFINITY; });
    say([](auto &l) { l.n_kv = 0; });
    say([](auto &l) { l.page_size = 48; });
    say([](auto &l) { l.page_size = 256; });
    say([](auto &l) { l.head_dim = 96; });
    say([](auto &l) { l.n_kv = 65536; });""")
    assert got == ["0"] * 3 + ["1"] * 12 + ["7"] * 4


def test_reference_block():
    x = np.zeros((1, 32))
    x[0, :4] = [12.0, -3.0, 0.5, -0.4]
    x[0, 16:19] = [2688.0, 5000.0, -5000.0]
    code, byte = ref.quantize(x)
    assert ref.e4m3_values()[byte[0, 0]] == 2.0 and ref.e4m3_values()[byte[0, 1]] == 448.0
    assert list(ref.values(code, byte)[0, :4]) == [12.0, -3.0, 0.0, -0.0]  # 0.25 and 0.2: to 0
    assert list(ref.values(code, byte)[0, 16:19]) == [2688.0, 2688.0, -2688.0]
    x[0, 20] = np.nan
    assert np.isnan(ref.values(*ref.quantize(x))[0, 16:]).all()
    assert ref.e4m3_values()[1] == 2.0 ** -9 and ref.e4m3_values()[8] == 2.0 ** -6 and ref.e4m3_values()[126] == 448


def test_reference_ties():
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    assert list(ref.GRID[ref.nearest(ties, ref.GRID)]) == [0, 1, 1, 2, 2, 4, 4]


@pytest.mark.parametrize("page,ring", [(16, 0), (64, 2)])
def test_reference_cache_round_trip(page, ring):
    rng = np.random.default_rng(0)
    c = ref.Cache(5, 2, 64, page, [[3, 1, 4, 0]], ring, 0.5, 2.0)
    rows = {p: (rng.standard_normal((2, 64)), rng.standard_normal((2, 64))) for p in range(40)}
    for p, (k, v) in rows.items():
        c.put(0, p, k, v)
    k, v = c.get(0, 40)
    for p, (a, b) in rows.items():
        assert np.array_equal(k[:, p], ref.values(*ref.quantize(a, 0.5), 0.5)) and np.array_equal(v[:, p], ref.values(*ref.quantize(b, 2.0), 2.0))


def test_reference_scores():
    x = np.log(np.array([0.5, 0.125, 0.25, 0.125]))
    lp, rank, ent, lse, ids, best = ref.scores(x, 3, 4)
    assert np.isclose(lp, np.log(0.125)) and rank == 3 and list(ids) == [0, 2, 1, 3] and np.isclose(ent, 1.75 * np.log(2)) and np.isclose(lse, 0)
