"""A norm kernel that needs more LDS than the device grants is not launched, and
its launcher says so: the launchers' own object, linked with an allow_lds that
refuses."""

from __future__ import annotations

import os
import shutil
import subprocess

import pytest

from rollfast_amd import build

SOURCE = """
#include "rf_norm_launch.h"

#include <cstdio>

rf_status rfb::allow_lds(const void*, size_t, std::atomic<uint64_t>&) noexcept { return RF_ERR_HIP; }

int main()
{
    rf_norm a{};  // 9000 columns, both norms: the kernel of broad rows
    a.rows = 1;
    a.cols = 9000;
    a.dtype = a.branch_dtype = RF_BF16;
    a.post = a.next = RF_NORM_RMS;
    rfb::NormShape s{};
    s.tpr = 576;
    s.ny = 1;
    s.nv = 2;
    const rfb::NormPlan p{1, 1};
    const rf_status got = rfb::norm_backward_1_1(a, s, p, nullptr, nullptr);
    std::printf("%d\\n", (int)got);
    return got == RF_ERR_HIP ? 0 : 1;
}
"""


def test_a_refused_lds_size_is_reported(tmp_path):
    obj = os.path.join(build.OBJ_DIR, "rf_norm_t1_u1.o")
    if not os.path.exists(obj) or shutil.which(build.HIPCC) is None:
        pytest.skip("needs hipcc and the built objects")
    src, main, out = (str(tmp_path / n) for n in ("t.hip", "t.o", "t"))
    with open(src, "w") as f:
        f.write(SOURCE)
    inc = [f"-I{build.CSRC}", f"-I{os.path.join(build.REPO, 'include')}"]
    for cmd in ([build.HIPCC, *build.FLAGS, *inc, "-c", src, "-o", main],
                [build.HIPCC, f"--offload-arch={build.ARCH}", main, obj, "-o", out], [out]):
        r = subprocess.run(cmd, capture_output=True, text=True, timeout=120)
        assert r.returncode == 0, r.stdout + r.stderr
