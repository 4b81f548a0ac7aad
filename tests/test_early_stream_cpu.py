"""What a context lets a decode launch read ahead of the launches in front of it, on the host: the bookkeeping of
csrc/internal.hpp against a model of which launches can still be in flight."""
import subprocess
from pathlib import Path

import pytest

SRC = Path(__file__).resolve().parent.parent / "test-burn_b200" / "csrc"

# A launch: plain (with or without writes to pools) or with the attribute.  In flight at the start of launch m: everything from
# the last strict launch on, or from the last plain one on, whichever is later (a strict launch has waited for all before it; a
# plain one starts when all before it are over; a relaxed one shows nothing).
PROGRAM = r"""
#include "internal.hpp"
#include <cstdio>
#include <cstdlib>
#include <vector>
struct Launch { bool plain, strict; int writes; };  // writes: cache number, -1 none, -2 any
int main()
{
    srand(7);
    int early = 0, held = 0;
    static char caches[16];
    for (int trial = 0; trial < 2000; ++trial) {
        MfContext ctx;
        std::vector<Launch> log;
        for (int m = 0; m < 40; ++m) {
            const int kind = rand() % 8, cache = rand() % 6;
            if (kind == 0 || kind == 1) {
                ctx.note_plain_launch(kind == 0);
                log.push_back({true, false, kind == 0 ? -2 : -1});
                continue;
            }
            const void *k = &caches[2 * cache], *v = &caches[2 * cache + 1];
            const bool may = ctx.may_stream_early(k, v), strict = ctx.next_launch_strict();
            bool hit = false;
            for (int i = (int)log.size() - 1; i >= 0; --i) {
                hit |= log[i].writes == cache || log[i].writes == -2;
                if (log[i].plain || log[i].strict) break;
            }
            if (may && hit) { printf("trial %d launch %d streams a cache that is being written\n", trial, m); return 1; }
            (may ? early : held) += 1;
            const bool append = rand() % 4 != 0;
            ctx.note_programmatic_launch(strict, append ? k : nullptr, append ? v : nullptr);
            log.push_back({false, strict, append ? cache : -1});
        }
    }
    printf("%d early, %d held\n", early, held);
    return early > 10000 && held > 1000 ? 0 : 2;
}
"""


def test_no_cache_is_streamed_while_it_is_written(tmp_path):
    cuda = Path("/usr/local/cuda/include")
    if not cuda.exists():
        pytest.skip("no CUDA headers")
    (tmp_path / "early.cpp").write_text(PROGRAM)
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-c", f"-I{SRC}", f"-I{cuda}", str(tmp_path / "early.cpp"),
                        "-o", str(tmp_path / "early.o")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run(["g++", str(tmp_path / "early.o"), "-o", str(tmp_path / "early")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([str(tmp_path / "early")], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
