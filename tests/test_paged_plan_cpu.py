"""The division of a paged attention launch among its blocks, run on the host from the kernel's own source."""
import os
import random
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "diffusers-tpu_b200", "csrc")


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    folder = tmp_path_factory.mktemp("plan")
    for name in ("paged.cuh", "paged_plan.cuh"):
        shutil.copy(os.path.join(CSRC, name), folder)
    for name in ("ptx.cuh", "plan.cc"):
        shutil.copy(os.path.join(HERE, "host_plan", name), folder)
    exe = str(folder / "plan")
    subprocess.run(["g++", "-std=c++20", "-O1", "-Wno-unknown-pragmas", "-fsanitize=undefined", "-fno-sanitize-recover", "-o", exe,
                    str(folder / "plan.cc"), "-lpthread"], check=True)
    return exe


def _line(new, kv, *, causal=1, window=0, tokens=64, Hkv=8, blocks=148, capacity=None, starts=None):
    starts = [sum(new[:i]) for i in range(len(new) + 1)] if starts is None else starts
    capacity = max(kv + [0]) if capacity is None else capacity
    return " ".join(map(str, [causal, window, tokens, Hkv, blocks, capacity, max(sum(new), 1), len(new), *starts, *kv]))


def _run(program, lines):
    r = subprocess.run([program], input="\n".join(lines) + "\n", capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    out = r.stdout.strip().splitlines()
    assert len(out) == len(lines)
    return out


def test_every_key_tile_is_swept_once(program):
    rng = random.Random(0)
    lines = [
        _line([1], [1]), _line([0], [5]), _line([0, 0], [0, 0]), _line([1, 0, 3], [0, 9, 2]), _line([1], [131072], Hkv=1), _line([1] * 4, [900, 200, 350, 1000]),
        _line([2048], [61234], tokens=50), _line([9360], [48872], causal=0, tokens=256, Hkv=40), _line([5000], [5000], tokens=64, Hkv=2),
        _line([40, 50], [30, 50]), _line([20000], [20000], window=300, Hkv=1), _line([3000, 1, 1, 1], [60000] * 4, window=5000, tokens=2, Hkv=1),
        _line([1] * 400, [rng.randint(0, 3000) for _ in range(400)]), _line([1] * 1000, [1] * 1000, Hkv=24),
        _line([1] * 200 + [1], [1] * 200 + [100000], Hkv=1), _line([65536], [65536], tokens=2, Hkv=1),
        _line([3, 3, 3], [40, 50, 60], starts=[-4, 2, 100, 6]), _line([3, 3], [2 ** 31 - 1, -5], capacity=1024), _line([4096] * 3, [70000, 9000, 40000], tokens=32),
        _line([1], [2 ** 31 - 1], capacity=2 ** 31 - 1024, Hkv=2), _line([4096], [2 ** 30], capacity=2 ** 31 - 1024, Hkv=100, tokens=2),
    ]
    for _ in range(60):
        B = rng.choice([1, 2, 5, 33, 90])
        kv = [int(2 ** rng.uniform(0, 16)) for _ in range(B)]
        new = [rng.choice([0, 1, 1, rng.randint(1, 300), min(n, 3000)]) for n in kv]
        causal = rng.random() < 0.8
        lines.append(_line(new, kv, causal=int(causal), window=rng.choice([0, 0, 1, 77, 4000]) if causal else 0, tokens=rng.choice([2, 10, 50, 64, 256]),
                           Hkv=rng.choice([1, 3, 8]), blocks=rng.choice([148, 148, 160, 7, 1])))
    _run(program, lines)


def test_blocks_get_equal_shares(program):
    """The heaviest block of a launch that has enough to do, against a 148th of everything."""
    lines = [_line([1] * 48, [2000 + 640 * i for i in range(48)]), _line([2048], [61234], tokens=50),
             _line([9360], [48872], causal=0, tokens=256, Hkv=40), _line([30000], [30000], tokens=64), _line([1], [131072], Hkv=8)]
    for line in _run(program, lines):
        words = line.replace(",", "").split()
        heaviest, total = int(words[words.index("block") + 1]), int(words[words.index("of", words.index("block")) + 1])
        assert heaviest <= 1.06 * total / 148 + 5, line
