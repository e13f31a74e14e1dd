"""The places that the shared-prefix plan counts (``prefix_decode.hip``): one workgroup of eight waves or four of two
per CU.  The built library's own code objects say what every instance needs: at most 256 registers a wave (two
waves per SIMD) and a share of the CU's 160 KB LDS."""
import pathlib
import re
import shutil
import struct
import subprocess

import pytest

from tq4_decode import build

READELF = shutil.which("llvm-readelf") or "/opt/rocm/llvm/bin/llvm-readelf"
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def code_objects():
    """The gfx950 code objects in the library's offload bundles."""
    data = build.LIB.read_bytes()
    for at in (m.start() for m in re.finditer(re.escape(MAGIC), data)):
        count, = struct.unpack_from("<Q", data, at + len(MAGIC))
        if not 0 < count < 16:
            continue  # the magic inside some other string
        pos = at + len(MAGIC) + 8
        for _ in range(count):
            offset, size, length = struct.unpack_from("<QQQ", data, pos)
            name = data[pos + 24:pos + 24 + length]
            pos += 24 + length
            if b"gfx950" in name and size:
                yield data[at + offset:at + offset + size]


def kernels(tmp_path):
    """{kernel name: (registers, LDS bytes)} of the library."""
    found = {}
    for i, obj in enumerate(code_objects()):
        path = tmp_path / f"{i}.co"
        path.write_bytes(obj)
        notes = subprocess.run([READELF, "--notes", str(path)], check=True, capture_output=True, text=True).stdout
        for text in re.split(r"\n\s+- \.agpr_count", notes)[1:]:
            field = lambda n: int(re.search(rf"\.{n}:\s+(\d+)", text).group(1))  # noqa: E731
            name = re.search(r"\.name:\s+(\S+)", text).group(1)
            agprs = int(re.match(r":\s+(\d+)", text).group(1))
            vgprs = field("vgpr_count")  # (with AGPRs, counted from the next multiple of 4)
            found[name] = (vgprs if agprs == 0 or vgprs > 256 else -(-vgprs // 4) * 4 + agprs, field("group_segment_fixed_size"))
    return found


@pytest.mark.skipif(not pathlib.Path(READELF).exists(), reason="needs llvm-readelf")
def test_every_instance_fits_its_places(tmp_path):
    if not build.LIB.exists():
        build.build()
    seen = set()
    for name, (registers, lds) in kernels(tmp_path).items():
        form = re.search(r"prefix_kernelILi\dELb\dELb\dELb\dELi(\d)ELi(\d)ELb", name)
        if not form:
            continue
        wr, wt = map(int, form.groups())
        seen.add((wr, wt))
        assert registers <= 256, (name, registers)
        assert lds * (1 if wr == 4 else 4) <= 160 * 1024, (name, lds)
    assert seen == {(4, 2), (2, 1)}
