"""The walk over the tiles of an orthogonalisation's rounds, no GPU."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_every_part_of_every_tile_is_one_items_and_nothing_lies_behind_the_last(tmp_path):
    exe = str(tmp_path / "ortho_walk")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", os.path.join(ROOT, "glades-ml_b200", "csrc"),
                    os.path.join(ROOT, "tests", "host", "ortho_walk.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
