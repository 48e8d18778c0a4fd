"""The cases of ``int8_plan_cases`` take the kernels that they name, and leave
none out.  Built with g++ from the header that the library plans with."""
import shutil
import subprocess
from pathlib import Path

import pytest

from drama_moe import _lib
from int8_plan_cases import GATED, PRODUCTS, T64

ROOT = Path(__file__).resolve().parents[1]
HIP = Path("/opt/rocm/include/hip/hip_runtime.h")


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    if shutil.which("g++") is None or not HIP.is_file():
        pytest.skip("needs g++ and the HIP headers")
    exe = tmp_path_factory.mktemp("plans") / "int8_plans"
    subprocess.run(["g++", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-w", "-I", str(HIP.parents[1]), "-I",
                    str(ROOT / "drama3-studio_amd" / "csrc"), str(ROOT / "tests" / "int8_plans.cpp"), "-o", str(exe)], check=True)

    def run(sizes):
        text = "".join(" ".join(str(v) for v in s) + "\n" for s in sizes)
        out = subprocess.run([str(exe)], input=text, capture_output=True, text=True, timeout=60, check=True).stdout
        return [tuple(map(int, line.split())) for line in out.splitlines()]
    return run


def test_each_case_takes_its_kernel(plans):
    got = plans([(rows, n, k, 0) for rows, k, n, _, _ in PRODUCTS] + [(rows, i, k, 1) for rows, k, i, _, _, _ in GATED])
    want = [c[-2:] for c in PRODUCTS + GATED]
    wrong = [(c, g) for c, g, w in zip(PRODUCTS + GATED, got, want) if g != w]
    assert not wrong


def test_the_cases_leave_no_kernel_out(plans):
    """Over a grid of sizes the plan names nothing that the cases do not."""
    sizes = [(rows, n, k) for rows in (1, 4, 16, 33, 64, 65, 128, 200, 513, 1100, 1300, 2048, 4100, 9000)
             for n in (64, 700, 2048, 2752, 4096, 5632, 11008, 12288, 33000) for k in (128, 1000, 4096, 5200, 7700, 10300, 16384)]
    for gated, cases in ((0, PRODUCTS), (1, GATED)):
        have = {c[-2:] for c in cases}
        assert set(plans([(*s, gated) for s in sizes])) <= have


@pytest.mark.parametrize("case", [c for c in PRODUCTS if c[-2] == T64] + [c for c in GATED if c[-2] == T64])
def test_shares_of_k_show_in_the_workspace(case):
    rows, k, n, *rest, _, splits = case
    gated = bool(rest)
    lib = _lib.library()
    rows8 = -(-(rows * (-(-k // 128) * 128 + 4)) // 256) * 256
    part = 4 * splits * rows * -(-n // 8) * 8 * (2 if gated else 1) if splits > 1 else 0
    if gated:
        hidden = -(-(rows * n * 4) // 256) * 256
        got = lib.dmoe_int8_feed_forward_workspace_bytes(rows, rest[0], k, n, _lib.F32)
        assert got == hidden + rows8 + part
    else:
        assert lib.dmoe_int8_linear_workspace_bytes(rows, n, k, 0) == rows8 + part
