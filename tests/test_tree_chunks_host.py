"""How positions over a paged cache are dealt to workgroups
(csrc/tree_chunks.h, no GPU): chunks by the launch rule, and the table entries
that a workgroup loads ahead, for every chunk length, place and page size."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <stdio.h>
#include <initializer_list>
#include "tree_chunks.h"

static unsigned pages(uint32_t key0, uint32_t n, uint32_t log) { return ((key0 + n - 1) >> log) - (key0 >> log) + 1; }

int main() {
    unsigned short_of = 0, past = 0, tight = 0, wrong = 0;
    // A chunk starts at a multiple of its length behind a multiple of STEP.
    for (uint32_t log = 2; log <= 10; log++)
        for (uint32_t chunk = STEP; chunk <= MAX_CHUNK; chunk += STEP)
            for (uint32_t base = 0; base <= 2048; base += STEP)
                for (uint32_t k = 0; k < 40; k++) {
                    const uint32_t key0 = base + k * chunk;
                    for (uint32_t n : {1u, chunk / 2, chunk - 1, chunk}) {
                        short_of += pages(key0, n, log) > most_pages(chunk, log);
                        past += pages(key0, n, log) > CHUNK_PAGES;
                    }
                    tight += pages(key0, chunk, log) == most_pages(chunk, log);
                }
    for (uint64_t pairs : {1ull, 2ull, 8ull, 31ull, 32ull, 100ull, 512ull, 1024ull, 4000ull, 65535ull})
        for (uint64_t span = 1; span <= 1u << 20; span += span / 7 + 1) {
            const uint32_t c = chunk_positions(span, pairs);
            wrong += c % STEP != 0 || c < STEP || c > MAX_CHUNK;
            // As many workgroups as wanted, unless the chunks are at their longest.
            wrong += c < MAX_CHUNK && (span + c - 1) / c > (1024 / pairs > 1 ? 1024 / pairs : 1);
        }
    printf("short %u past %u wrong %u tight %d\n", short_of, past, wrong, tight > 0);
    return 0;
}
"""


def test_entries_loaded_ahead_cover_every_chunk(tmp_path):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no host compiler")
    src, exe = tmp_path / "chunks.cpp", tmp_path / "chunks"
    src.write_text(PROGRAM)
    subprocess.run([cxx, "-std=c++17", "-O2", "-Wall", "-Werror", "-I", os.path.join(ROOT, "iris_amd", "csrc"), str(src), "-o",
                    str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=100)
    assert r.stdout == "short 0 past 0 wrong 0 tight 1\n"
