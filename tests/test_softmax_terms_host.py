"""The softmax's exp terms in double arithmetic (csrc/softmax_double.h, no GPU)
against the oracle's integers: every difference that has a non-zero term, and
larger ones to the end of the range."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <stdio.h>
#include "detnum.h"
#include "softmax_double.h"

static int differs(uint32_t diff) {
    uint32_t kept;
    const int64_t want = dn_softmax_exp_term(-(int64_t)diff * 65536);
    const double got = softmax_term(diff, &kept);
    return got != (double)want || kept != (diff ? (uint32_t)want : 0xffffffffu);
}

int main(void) {
    unsigned bad = 0;
    for (uint32_t d = 0; d <= 1u << 21; d++) bad += differs(d);
    for (uint64_t d = 1u << 21; d <= 0xffffffffu; d += 65521) bad += differs((uint32_t)d);
    bad += differs(0x7fffffffu) + differs(0x80000000u) + differs(0xffffffffu);
    printf("%u\n", bad);
    return bad != 0;
}
"""


@pytest.mark.parametrize("flags", [["-O0"], ["-O2", "-mfma"]])
def test_terms_are_the_integers(tmp_path, flags):
    cc = shutil.which("gcc")
    if cc is None:
        pytest.skip("no host compiler")
    if "-mfma" in flags and "fma" not in open("/proc/cpuinfo").read():
        pytest.skip("no fused multiply-add here")
    src, exe = tmp_path / "terms.c", tmp_path / "terms"
    src.write_text(PROGRAM)
    oracle = os.path.join(ROOT, "oracle")
    subprocess.run([cc, "-std=gnu11", *flags, "-ffp-contract=off", "-I", oracle, "-I", os.path.join(ROOT, "iris_amd", "csrc"),
                    str(src), os.path.join(oracle, "detnum.c"), "-lm", "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stdout
