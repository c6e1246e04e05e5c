"""Host-side parts of the 4-bit operators that need no GPU."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_a_failed_capacity_query_is_asked_again(tmp_path):
    """Answers 0, -1, 7: the failures are returned and not kept, the 7 is (a fourth question would get a 9)."""
    exe = str(tmp_path / "kept_test")
    subprocess.run([os.environ.get("CXX", "g++"), "-std=c++17", "-O1", "-pthread", os.path.join(ROOT, "tests", "csrc", "kept_test.cpp"), "-o", exe], check=True)
    out = subprocess.run([exe], check=True, capture_output=True, text=True, timeout=60).stdout
    assert out.split() == ["0/1", "-1/2", "7/3", "7/3", "7/3", "0"]
