"""The embedding's kernels (burn_dragon_amd/csrc/embed.hip), compiled for the CPU
(tests/simt) and run between pages that nothing may touch: every access of the
lookup, the sort, the clears, the sums and their joins lies in its buffer, for
tails of columns, runs and workgroups of all kinds, and the results are the
formula's."""
import os
import platform
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _clang():
    for cand in ("/opt/rocm/llvm/bin/clang++", "/opt/rocm/bin/amdclang++"):
        if os.path.exists(cand):
            return cand
    return None


@pytest.fixture(scope="module")
def on_cpu(tmp_path_factory):
    clang = _clang()
    if clang is None or platform.machine() != "x86_64":
        pytest.skip("no clang for x86-64")
    simt, exe = os.path.join(ROOT, "tests", "simt"), str(tmp_path_factory.mktemp("simt") / "embed_on_cpu")
    r = subprocess.run([clang, "-x", "c++", "-std=c++17", "-O1", "-w", f"-I{simt}",
                        f"-I{os.path.join(ROOT, 'burn_dragon_amd', 'csrc')}", f"-I{os.path.join(ROOT, 'include')}",
                        os.path.join(simt, "embed_on_cpu.cc"), "-o", exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]

    def one(case):
        r = subprocess.run([exe] + [str(a) for a in case], capture_output=True, text=True, timeout=120)
        return r.returncode, (case, r.stdout + r.stderr)

    def run(cases):
        """(exit status, (case, output)) of each (op, n, V, D, bf16, norm, accumulate, kind, front)."""
        with ThreadPoolExecutor(max_workers=6) as ex:
            return list(ex.map(one, cases))
    return run


DIMS = [1, 3, 4, 7, 8, 63, 64, 65, 200, 256, 257, 511, 512, 1000, 1024, 1027, 2047, 2048]


@pytest.mark.parametrize("D", DIMS)
def test_columns(on_cpu, D):
    # 333 tokens go by the sort, 40 without.
    for rc, text in on_cpu([(*case, "uniform", front) for bf16 in (0, 1) for norm in (0, 1) for front in (0, 1) for case in (
            ("embed", 37, 11, D, bf16, norm, 0), ("vjp", 333, 50, D, bf16, norm, front),
            ("vjp", 40, 13, D, bf16, norm, 1 - front))]):
        assert rc == 0, text


@pytest.mark.parametrize("n,V,D", [(1, 1, 5), (2, 300, 4), (63, 7, 9), (64, 1, 8), (65, 3, 12), (129, 511, 20),
                                   (1023, 512, 5), (4096, 9, 3), (4097, 300, 6), (5121, 70000, 2), (9001, 256, 33),
                                   (300, 262143, 1), (2000, 262144, 1)])
def test_tokens(on_cpu, n, V, D):
    for rc, text in on_cpu([(*case, kind, front) for kind in ("uniform", "few", "one") for front in (0, 1) for case in (
            ("vjp", n, V, D, 0, 0, front), ("vjp", n, V, D, 1, 1, 1 - front))]):
        assert rc == 0, text


def test_many_tokens(on_cpu):
    # Longer runs; four rounds a workgroup.
    for rc, text in on_cpu([(*case, n % 2) for n in (16384, 32769, 131073) for case in (
            ("vjp", n, 300, 4, 0, 1, 0, "uniform"), ("vjp", n, 4000, 3, 0, 0, 1, "few"),
            ("embed", n, 300, 5, 1, 1, 0, "uniform"))]):
        assert rc == 0, text


@pytest.mark.parametrize("op", ["embed", "vjp"])
def test_an_access_out_of_range_is_noticed(on_cpu, op):
    # The last row of the table (of the gradient) is not there.
    for rc, text in on_cpu([(op, n, 5, D, 0, 0, 0, "short", 0) for n in (40, 333) for D in (64, 2047)]):
        assert rc == 5 and "out of range" in text[1], text
