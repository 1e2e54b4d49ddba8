"""Every gfx950 code object of the built libraries against the two MFMA rules that the compiler keeps for its own instructions alone
(tests/test_code_hazards.py states them and has the walks): a VALU write of a VGPR and an MFMA that reads it two wait states on, an MFMA
that reads a VGPR as C and a VALU write of it three on. A library holds one object a source file, in bundles one after another in its
.hip_fatbin section; that file's own walks over a library read the first one (the trellis kernels, whose guard it holds as well).
An inline-asm block's outputs are what the compiler does not see, so these walks are what keeps a new one out of MFMA operands."""
import os
import shutil
import struct
import subprocess

import pytest

from test_code_hazards import LLVM, ROOT, violations, war_violations

MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"
PKG = os.path.join(ROOT, "radiance-exl3_amd")
# the kernels that name each object, and the least MFMAs it holds
OBJECTS = {"libexl3c4.so": {"k_gu_pf": 1000, "k_mg_tile": 1000, "k_mx4_quant": 0, "k_router": 0},
           "libexl3c4_calib.so": {}}


def objects(fat):
    """The gfx950 code objects of a .hip_fatbin section: its bundles, each a count, then (offset, size, target) of its entries."""
    at = fat.find(MAGIC)
    while at >= 0:
        n, = struct.unpack_from("<Q", fat, at + 24)
        p = at + 32
        for _ in range(n):
            off, size, length = struct.unpack_from("<QQQ", fat, p)
            target = fat[p + 24:p + 24 + length].decode()
            p += 24 + length
            if target.endswith("gfx950") and size:
                yield fat[at + off:at + off + size]
        at = fat.find(MAGIC, at + 24)


def with_scales(lines):
    """The lines with each scaled MFMA's two scale registers in the place of its A and B, for the same walk."""
    for l in lines:
        if "v_mfma_scale" in l and "//" in l:
            op, rest = l.split("//")[0].strip().split(" ", 1)
            a = [t.strip() for t in rest.split(",")]
            l = f"\t{op} {a[0]}, {a[4].split()[0]}, {a[5].split()[0]}, {a[3]} // "
        yield l


@pytest.fixture(scope="module", params=list(OBJECTS))
def listing(request, tmp_path_factory):
    """(library, each object's disassembly)."""
    lib = os.path.join(PKG, request.param)
    tools = [os.path.join(LLVM, t) for t in ("llvm-objcopy", "llvm-objdump")]
    if not os.path.exists(lib):
        pytest.skip(f"{request.param} is not built")
    if not all(shutil.which(t) for t in tools):
        pytest.skip("the ROCm LLVM tools are not installed")
    tmp = tmp_path_factory.mktemp("objects")
    fat, out = str(tmp / "fat.bin"), []
    subprocess.run([tools[0], f"--dump-section=.hip_fatbin={fat}", lib, str(tmp / "lib.so")], check=True)
    with open(fat, "rb") as f:
        found = list(objects(f.read()))
    for i, o in enumerate(found):
        path = str(tmp / f"{i}.o")
        with open(path, "wb") as f:
            f.write(o)
        out.append(subprocess.run([tools[1], "-d", "--mcpu=gfx950", path], check=True, capture_output=True, text=True).stdout.splitlines())
    return request.param, out


def test_every_object_is_read(listing):
    """Each source file's kernels are in one of the objects, with the MFMAs it has at least."""
    lib, objs = listing
    assert len(objs) >= max(1, len(OBJECTS[lib]))
    for kernel, least in OBJECTS[lib].items():
        mine = [o for o in objs if any(l.endswith(">:") and kernel in l for l in o)]
        assert len(mine) == 1, kernel
        assert sum(l.strip().startswith("v_mfma") for l in mine[0]) >= least, kernel


def test_no_mfma_reads_a_fresh_write_or_loses_its_c(listing):
    lib, objs = listing
    for o in objs:
        raw, war = violations(o) + violations(list(with_scales(o))), war_violations(o)
        for v in raw[:5] + war[:5]:
            print(" | ".join(map(str, v)))
        assert not raw and not war, f"{lib}: {len(raw)} fresh reads, {len(war)} writes of a C that is being read"


def test_the_scales_of_an_mfma_are_seen():
    """A VALU write of a scale register right before the scaled MFMA (too soon), and two wait states before it."""
    f = "0000 <k>:"
    mf = "\tv_mfma_scale_f32_16x16x128_f8f6f4 v[10:13], v[44:47], v[48:51], v[10:13], v60, v61 op_sel_hi:[0,0,0] cbsz:4 blgp:4 // 0: 1"
    for r in (60, 61):
        assert len(violations(list(with_scales([f, f"\tv_mov_b32_e32 v{r}, v1 // 0: 1", mf])))) == 1
        assert violations(list(with_scales([f, f"\tv_mov_b32_e32 v{r}, v1 // 0: 1", "\ts_nop 1 // 0: 1", mf]))) == []
    assert len(violations([f, "\tv_mov_b32_e32 v48, v1 // 0: 1", mf])) == 1
