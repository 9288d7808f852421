"""CPU replay of the attention rows' loop (tests/rows_schedule_check.cpp): no instance reads a
fragment that its loads were not waited for, or loads over one that is still read."""
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]


def replay(tmp_path, *flags):
    exe = tmp_path / "rows_schedule_check"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", *flags, f"-I{ROOT / 'welder_typical_chain_amd' / 'csrc'}",
                    str(ROOT / "tests" / "rows_schedule_check.cpp"), "-o", str(exe)], check=True)
    return subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)


def test_every_instance_waits_for_what_it_reads(tmp_path):
    res = replay(tmp_path)
    assert res.returncode == 0, res.stdout + res.stderr
    assert res.stdout.strip().splitlines()[-1] == "OK"


def test_the_replay_sees_loads_behind_the_wait(tmp_path):
    res = replay(tmp_path, "-DLATE")
    assert res.returncode == 1 and "PREFIX 1 A 1" in res.stdout and "read before it landed" in res.stdout


def test_such_an_order_does_not_compile(tmp_path):
    csrc = ROOT / "welder_typical_chain_amd" / "csrc"
    text = (csrc / "rows_schedule.h").read_text()
    changed = text.replace("A == 1 && !(PREFIX && ND == 1) ? 4 : 3", "A == 1 ? 4 : 3")
    assert changed != text
    (tmp_path / "rows_schedule.h").write_text(changed)
    res = subprocess.run(["g++", "-std=c++17", "-fsyntax-only", f"-I{tmp_path}", str(ROOT / "tests" / "rows_schedule_check.cpp")],
                         capture_output=True, text=True)
    assert res.returncode != 0 and "before the wait that counts them" in res.stderr
