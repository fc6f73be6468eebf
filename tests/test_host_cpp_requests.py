"""The C++ mirror's adapters, expert block and rules on logits: the demo program runs them beside the C calls that they stand for, bit for bit."""
import subprocess

import pytest

from tests.test_host_cpp import build_demo


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ["9", "32", "70"])
def test_mirror_of_the_request_operators(tmp_path, rows):
    r = subprocess.run([build_demo(tmp_path), rows, "512", "768", "3"], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "request operators equal the C calls: yes" in r.stdout
