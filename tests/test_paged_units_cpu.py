"""The units that a block of a paged attention launch takes, in the order in which its warps take them, from the kernel's own source."""
import os
import random
import shutil
import subprocess

import pytest

from test_paged_plan_cpu import CSRC, HERE, _line


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    folder = tmp_path_factory.mktemp("units")
    for name in ("paged.cuh", "paged_plan.cuh"):
        shutil.copy(os.path.join(CSRC, name), folder)
    for name in ("ptx.cuh", "units.cc"):
        shutil.copy(os.path.join(HERE, "host_plan", name), folder)
    exe = str(folder / "units")
    subprocess.run(["g++", "-std=c++20", "-O1", "-Wno-unknown-pragmas", "-fsanitize=undefined", "-fno-sanitize-recover", "-o", exe,
                    str(folder / "units.cc"), "-lpthread"], check=True)
    return exe


def _run(program, lines):
    r = subprocess.run([program], input="\n".join(lines) + "\n", capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    return [(int(line.split()[0]), int(line.split()[2])) for line in r.stdout.strip().splitlines()]


def test_long_prompts_of_many_rounds(program):
    """Prompts of which every block is dealt 16 whole units and more: the range behind them begins in the middle of a unit, and the
    warp that describes the units behind the first 16 has to say so."""
    found = _run(program, [_line([16384], [16384], tokens=50), _line([16384], [16384], tokens=256, Hkv=40), _line([8192] * 3, [8192] * 3, tokens=50),
                           _line([32768], [32768], tokens=64), _line([20000], [90000], tokens=64, window=30000), _line([9000, 1, 20000], [9000, 70, 25000], tokens=32)])
    assert any(rounds >= 16 and behind > 50 for rounds, behind in found), found


def test_units_of_mixed_batches(program):
    rng = random.Random(1)
    lines = [_line([1] * 400, [rng.randint(0, 3000) for _ in range(400)]), _line([1, 0, 3], [0, 9, 2]), _line([65536], [65536], tokens=2, Hkv=1)]
    for _ in range(30):
        kv = [int(2 ** rng.uniform(0, 15)) for _ in range(rng.choice([1, 3, 40]))]
        new = [rng.choice([0, 1, rng.randint(1, 300), min(n, 6000)]) for n in kv]
        causal = rng.random() < 0.8
        lines.append(_line(new, kv, causal=int(causal), window=rng.choice([0, 0, 77, 4000]) if causal else 0, tokens=rng.choice([2, 10, 64, 256]),
                           Hkv=rng.choice([1, 3, 8]), blocks=rng.choice([148, 160, 7, 1])))
    _run(program, lines)


def test_starts_out_of_order_do_not_overflow_the_units(tmp_path):
    """Starts that go up and down give the same rows to many sequences: more units than an int can number are none."""
    for name in ("paged.cuh", "paged_plan.cuh"):
        shutil.copy(os.path.join(CSRC, name), tmp_path)
    for name in ("ptx.cuh", "cuts.cc"):
        shutil.copy(os.path.join(HERE, "host_plan", name), tmp_path)
    subprocess.run(["g++", "-std=c++20", "-O1", "-Wno-unknown-pragmas", "-fsanitize=undefined", "-fno-sanitize-recover", "-o", str(tmp_path / "cuts"),
                    str(tmp_path / "cuts.cc"), "-lpthread"], check=True)

    def line(B, T, tokens, Hkv):
        return _line([0] * (B - 1) + [T], [50] * B, tokens=tokens, Hkv=Hkv, starts=[b % 2 * T for b in range(B + 1)])

    calls = [line(8192, 1 << 20, 2, 1), line(8192, 1 << 20, 256, 128), line(8192, 1 << 30, 2, 1), line(64, 1000, 2, 1)]
    out = subprocess.run([str(tmp_path / "cuts")], input="\n".join(calls) + "\n", capture_output=True, text=True, timeout=100, check=True).stdout
    found = [tuple(map(int, x.split())) for x in out.split("\n") if x]
    assert found == [(-1, 0), (-1, 0), (-1, 0), (0, 32 * 500)], found
