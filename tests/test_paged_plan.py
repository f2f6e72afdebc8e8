"""The paged attention's arithmetic on numbers that lie on the device, and how much its launches take (paged_plan.hpp),
compiled for the host: whatever the numbers, what becomes an address stays inside its buffer."""
import random
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
HDR = ROOT / "llamd_rs_amd" / "csrc" / "paged_plan.hpp"


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    exe = tmp_path_factory.mktemp("paged_plan") / "paged_plan"
    subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", f"-I{HDR.parent}", "-o", str(exe),
                    str(ROOT / "tests" / "native" / "paged_plan.cpp")], check=True)

    def run(lines):
        done = subprocess.run([str(exe)], input="\n".join(lines), capture_output=True, text=True)
        assert done.returncode == 0, done.stderr
        return [tuple(int(x) for x in line.split()) for line in done.stdout.splitlines()]
    return run


def test_shared_positions_stay_in_the_table(plan):
    """Any number on the device: whole pages, none past the table. A wave steps up to 127 positions past the shared ones, and a
    sequence of no positions does so without a test of its length before: 2^31 - 16 shared positions would wrap."""
    numbers = [-(1 << 31), -1, 0, 1, 15, 16, 17, 100, 4095, 4096, 1 << 30, (1 << 30) + 1, (1 << 31) - 64, (1 << 31) - 16, (1 << 31) - 1]
    cases = [(n, log, most) for n in numbers for log in range(4, 9) for most in (1, 3, 257, 1 << (30 - log))]
    for (n, log, most), (got,) in zip(cases, plan([f"shared {n} {log} {most}" for n, log, most in cases])):
        assert got == min(max(n, 0), most << log) >> log << log
        assert got + 128 < 1 << 31


def test_a_row_of_a_prefix_finds_a_slot(plan):
    """Starts of groups that go back to the first sequence again and again claim the whole batch each time: 100000 sequences
    of 64 heads, 50000 groups of 50001 tiles, 2.5e9 in all. Sums and slots stay in their ranges; groups that make sense keep
    their places."""
    cases = []
    for groups, more, tiles in ((100_000, 50_001, 150_000), (100_000, (1 << 22) - 1, (1 << 22) - 1), (3, 7, 9), (1, 1, 1), (0, 5, 5)):
        for row in (0, 127, 128, 6_399_999, (1 << 31) - 1):
            cases.append((groups, more, tiles, 128, row, 0))
    for (groups, more, tiles, R, row, _), (total, tile) in zip(cases, plan([f"join {' '.join(map(str, c))}" for c in cases])):
        assert 0 <= total <= 64 * tiles and 0 <= tile < tiles
        if (groups + 1) // 2 * more <= tiles:
            assert total == (groups + 1) // 2 * more and tile == min(total + row // R, tiles - 1)
    assert plan(["join 0 0 40 128 300 11"]) == [(0, 13)]


def test_tiles_and_parts_of_any_pieces(plan):
    """Rows cut into pieces anyhow never make more tiles than there are slots for, and slots stay within five times the
    workgroups wanted (tiles <= full tiles + pieces <= 5 max(full tiles, pieces / 4)), or the tiles themselves where these are
    more."""
    rng = random.Random(5)
    cases = []
    for R in (16, 128):
        for rows, pieces in ((8, 64), (1, 1), (64, 32), (2048, 512), (4096, 0), (12, 12), (100_000, 3), (1 << 20, 1 << 16)):
            cases += [(rows, pieces, R, kv, 512, most, 64) for kv in (1, 4, 32) for most in (0, 16, 4096)]
    for (rows, pieces, R, kv, want, most, cap), (tiles, parts) in zip(cases, plan([f"tiles {' '.join(map(str, c))}" for c in cases])):
        assert 1 <= parts <= max(1, min(most, cap))
        assert parts == 1 or tiles * kv * parts <= 5 * want
        for _ in range(4):
            cuts = sorted(rng.randrange(rows + 1) for _ in range(max(pieces, 1) - 1)) + [rows]
            sizes = [b - a for a, b in zip([0] + cuts, cuts)]
            if pieces:
                assert sum(-(-n // R) for n in sizes) <= tiles
    # 64 sequences in pairs, heads of their own; 48 sequences of 8 heads behind one prefix
    assert plan(["tiles 64 32 128 32 512 16 64", "tiles 384 1 128 4 512 9 64"]) == [(32, 2), (4, 9)]
