"""Code-generation checks of the 8-bit serving kernels (CPU only: hipcc cross-compiles
gfx950 and these tests read the AMD assembly of our own build)."""

from __future__ import annotations

import re
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

from pare_amd import build as B

SOURCES = ["paged_kv.hip", "paged_attention.hip", "w8a8.hip"]


@pytest.fixture(scope="module")
def asm(tmp_path_factory) -> dict[str, str]:
    try:
        cc = B._hipcc()
    except RuntimeError:
        pytest.skip("hipcc not available")
    out = tmp_path_factory.mktemp("asm")
    flags = [f for f in B.HIPCC_FLAGS if f not in ("-shared", "-fPIC")]

    def one(src: str) -> str:
        to = out / (src + ".s")
        res = subprocess.run([cc, *flags, f"-I{B.REPO_DIR / 'include'}", "--cuda-device-only", "-S",
                              str(B.CSRC / src), "-o", str(to)], capture_output=True, text=True)
        assert res.returncode == 0, res.stderr[-2000:]
        return to.read_text()

    with ThreadPoolExecutor() as pool:
        return dict(zip(SOURCES, pool.map(one, SOURCES)))


def test_no_64_bit_shift_by_a_vector_register(asm):
    """A 64-bit shift whose amount is in the last vector register of the wave's allocation has
    given wrong lanes (the attention of 16 query rows over e4m3 codes, 128 registers, v127):
    no kernel here shifts 64 bits by an amount of a lane's own."""
    for src, text in asm.items():
        found = re.findall(r"v_(?:lshl|lshr|ashr)rev_[bi]64\S* v\[\d+:\d+\], v\d+", text)
        assert not found, (src, found[:3])


def test_no_packed_fp32_and_no_spills(asm):
    for src, text in asm.items():
        assert not re.search(r"v_pk_(add|mul|fma)_f32", text), src
        spills = re.findall(r"^\s*; ScratchSize: (\d+)", text, re.M)
        assert spills and all(int(s) == 0 for s in spills), (src, spills)
