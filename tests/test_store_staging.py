"""How the writer's workgroups stage the rotation matrix (``csrc/store.h``), read from the compiler's listing: the
loads go out in the order in which the staging takes them, so that the first LDS writes stand while
the last loads are still on their way."""
import pathlib
import re
import shutil
import subprocess

import pytest

from tq4_decode import build

SOURCE = """
#include "{csrc}/store.h"
template __global__ void tq4::store::store_kernel<{layout}, __bf16, {kb}, 4, {waves}>(
    const __bf16 *, const __bf16 *, const int32_t *, const float *, const float *, const float *, uint8_t *, int, int, int,
    int64_t, int, int, int);
"""


def listing(tmp_path, **kw):
    src, out = tmp_path / "one.hip", tmp_path / "one.s"
    src.write_text(SOURCE.format(csrc=build.CSRC, **kw))
    flags = [f for f in build.HIPCC_FLAGS if f != "-fPIC"]
    subprocess.run([build.hipcc(), *flags, "-S", "--offload-device-only", "-o", str(out), str(src)], check=True, capture_output=True)
    body = re.search(r"^_Z\S*store_kernel\S*:.*?\n(.*?)\.Lfunc_end", out.read_text(), re.S | re.M)
    return [line.strip() for line in body.group(1).splitlines()]


@pytest.mark.skipif(not (shutil.which("hipcc") or pathlib.Path("/opt/rocm/bin/hipcc").exists()), reason="needs hipcc")
@pytest.mark.parametrize("layout,kb,waves", [(0, 4, 4), (1, 4, 4), (0, 3, 4), (0, 4, 8)])
def test_staging_starts_with_the_first_loads(tmp_path, layout, kb, waves):
    code = listing(tmp_path, layout=layout, kb=kb, waves=waves)
    steps = 128 * 16 // (64 * waves)  # of eight loads and two LDS writes
    first = next(i for i, line in enumerate(code) if line.startswith("ds_write_b128"))
    loads = sum(line.startswith("global_load_dword ") for line in code[:first])
    assert loads == 8 * steps
    waits = [int(n) for line in code[:first] for n in re.findall(r"vmcnt\((\d+)\)", line)]
    # all but the first step's loads (and K's and V's behind them) may still be on their way
    assert min(waits) >= min(8 * (steps - 1), 48), waits
