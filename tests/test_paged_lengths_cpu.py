"""Which keys a new token sees, lengths past what the page table can name among them, from the kernels' own source."""
import os
import random
import shutil
import subprocess

import pytest

from test_paged_plan_cpu import CSRC, HERE, _line


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    folder = tmp_path_factory.mktemp("seen")
    for name in ("paged.cuh", "paged_plan.cuh"):
        shutil.copy(os.path.join(CSRC, name), folder)
    for name in ("ptx.cuh", "seen.cc"):
        shutil.copy(os.path.join(HERE, "host_plan", name), folder)
    exe = str(folder / "seen")
    subprocess.run(["g++", "-std=c++20", "-O1", "-Wno-unknown-pragmas", "-fsanitize=undefined", "-fno-sanitize-recover", "-o", exe,
                    str(folder / "seen.cc"), "-lpthread"], check=True)
    return exe


def _seen(new, kv, causal, window, capacity):
    """Keys of each token.  A token has the slot that it was appended to; where the table has none for any new token of the
    sequence, the new ones count as its last."""
    out = []
    for n, m in zip(new, kv):
        end = min(max(m, 0), capacity)
        first = max(m, 0) - n
        if first >= capacity:
            first = capacity - n
        for i in range(n):
            slot = first + i
            out.append({j for j in range(end) if not causal or (j <= slot and (not window or j > slot - window))})
    return out


def test_tokens_see_what_is_in_front_of_their_slots(program):
    rng = random.Random(2)
    calls = [([10], [70], 1, 0, 64), ([10], [70], 1, 7, 64), ([10], [70], 0, 0, 64), ([10], [64], 1, 0, 64), ([4, 4], [2 ** 31 - 1, 50], 1, 0, 64),
             ([300, 1], [500, 65], 1, 40, 256), ([40, 50], [30, 50], 1, 0, 64), ([3, 3], [-5, 0], 1, 0, 16), ([1], [17], 1, 1, 16), ([5], [20], 1, 2, 16)]
    for _ in range(200):
        capacity = rng.choice([16, 64, 256])
        new = [rng.choice([0, 1, rng.randint(1, 90)]) for _ in range(3)]
        causal = rng.random() < 0.8
        calls.append((new, [rng.randint(0, 2 * capacity) for _ in new], int(causal), rng.choice([0, 0, 1, 9, 100]) if causal else 0, capacity))
    lines = [_line(new, kv, causal=causal, window=window, tokens=rng.choice([2, 10, 64]), capacity=capacity) for new, kv, causal, window, capacity in calls]
    r = subprocess.run([program], input="\n".join(lines) + "\n", capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stdout[-300:] + r.stderr
    for call, line in zip(calls, r.stdout.split("\n")):
        numbers = [int(x) for x in line.split()]
        assert [set(range(x, y)) for x, y in zip(numbers[::2], numbers[1::2])] == _seen(*call), call
