"""CPU: every size that the limits of i8_abi.h allow has a launch: fewer than 2^32 threads, which is what a grid may have."""
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def forms(tmp_path_factory):
    from nihilus_amd.build import hipcc

    out = str(tmp_path_factory.mktemp("forms") / "i8_forms")
    subprocess.run([hipcc(), "-x", "hip", "--cuda-host-only", "--offload-arch=gfx950", "-O1", "-std=c++20", "-I", os.path.join(ROOT, "include"), os.path.join(ROOT, "tests", "cpp", "i8_forms.cpp"), "-o", out],
                   check=True, capture_output=True)
    return lambda sizes: [tuple(map(int, line.split())) for line in subprocess.run([out], input="\n".join(" ".join(map(str, s)) for s in sizes), text=True, check=True, capture_output=True).stdout.splitlines()]


def test_no_launch_has_more_threads_than_a_grid_holds(forms):
    rng = random.Random(1)
    sizes = [(n, m, steps, behind) for e in range(19) for n in (1 << e, (1 << e) - 1 or 1) for m in {min(1 << 18, (1 << 30) // n), min(1 << 18, (1 << 30) // n) // 2 or 1} for steps in (1, 2, 16, 2047) for behind in (66, 78, 156)]
    for _ in range(2000):
        n = int(2 ** rng.uniform(0, 18))
        sizes.append((n, int(2 ** rng.uniform(0, min(18.0, 30 - n.bit_length()))), rng.choice((1, 2, 3, 8, 64)), rng.choice((66, 78, 156))))
    # (ceil(M / 256) ceil(N / 256) is up to 2^22)
    sizes = [s for s in sizes if (s[0] + 15) // 16 * ((s[1] + 15) // 16) <= 1 << 22]
    got = forms(sizes)
    assert len(got) == len(sizes) > 2000
    for size, (threads, form) in zip(sizes, got):
        assert threads < 1 << 32, (size, form)
