"""The check of what the paged attention's join finds in the plan's scratch, on the host (tests/cpp/join_record_test.cpp) with the header that the kernel
includes: no record of any bits leads outside the tensors."""
import pathlib
import subprocess

ROOT = pathlib.Path(__file__).resolve().parents[1]


def test_no_record_leads_outside(tmp_path):
    binary = tmp_path / "join_record_test"
    subprocess.run(["g++", "-O2", "-std=c++17", "-I", str(ROOT / "augur_v100_b200/csrc"), "-o", str(binary), str(ROOT / "tests/cpp/join_record_test.cpp")],
                   check=True, capture_output=True, text=True, timeout=120)
    done = subprocess.run([str(binary)], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0 and done.stdout.strip() == "ok", done.stdout
