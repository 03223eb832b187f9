"""Tests that have ended their process for a cause not found yet stay off, by file and name, and so does bench.py's use of the same loop."""
import os
import subprocess
import sys

import conftest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class _Item:
    def __init__(self, path, name):
        import pathlib

        self.path, self.originalname, self.name, self.marks, self.keywords = pathlib.Path(path), name, name + "[0]", [], {}

    def add_marker(self, m):
        self.marks.append(m)


def test_skips_go_by_file_and_name():
    for file, name in conftest.UNEXPLAINED_ABORTS:
        assert os.path.exists(os.path.join(ROOT, "tests", file))
        here, there = _Item(f"tests/{file}", name), _Item("tests/test_other_file.py", name)
        conftest.pytest_collection_modifyitems(None, [here, there])
        assert [m.name for m in here.marks].count("skip") == 1 and not there.marks


def test_bench_leaves_the_upload_loop_off():
    code = "import sys; sys.argv = ['bench.py']; import bench; print('upload', bench.parse_args([]).upload_variant)"
    out = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert "upload 0" in out.stdout, out.stderr[-2000:]
