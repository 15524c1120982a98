"""The rings of the prefill kernel over an 8-bit cache, one per padded head dim, on the CPU."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_every_ring_over_an_8_bit_cache(tmp_path):
    exe = str(tmp_path / "kv_raw_rings")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-I", os.path.join(ROOT, "scicompute_attention_b200", "csrc", "kernels"),
                    os.path.join(ROOT, "tests", "cpp", "kv_raw_rings.cpp"), "-o", exe], check=True)
    out = subprocess.run([exe], check=True, capture_output=True, text=True, timeout=120).stdout
    rows = {tuple(map(int, line.split()[:2])): tuple(map(int, line.split()[2:])) for line in out.splitlines()}
    assert len(rows) == 9
    for dim in (64, 128, 256):
        assert rows[dim, 0] == (0, 0), (dim, rows[dim, 0])
        assert sum(rows[dim, 1]) > 0 and sum(rows[dim, 2]) > 0, dim  # the model sees the mistakes
