"""Where the partials of an attention lie in its workspace, without a GPU: row numbers beyond 2^32."""
import os
import shutil
import subprocess

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"

PROGRAM = """
#include "attention.h"
#include <type_traits>
using kvc::attn::partial_row;
static_assert(std::is_same<decltype(partial_row(0, 1, 0, 16, 0)), int64_t>::value, "64 bits");
// 8191 narrow tiles of as many requests behind a shared prefix, 32768 key heads: 2^32 rows and more
static_assert(partial_row(8191, 32768, 32767, 16, 15) == (int64_t(1) << 32) - 1, "the last below");
static_assert(partial_row(8192, 32768, 0, 16, 0) == int64_t(1) << 32, "the first beyond");
static_assert(partial_row(8706, 32768, 5, 16, 3) == 8706 * int64_t(32768 * 16) + 5 * 16 + 3, "beyond");
static_assert(partial_row(1 << 20, 0xffff, 0xfffe, 128, 127) == ((int64_t(1) << 20) * 0xffff + 0xfffe) * 128 + 127, "wide tiles");
static_assert(partial_row(3, 2, 1, 16, 4) == 116, "small");
"""


def test_row_numbers_beyond_32_bits(tmp_path):
    if not os.path.exists(HIPCC):
        pytest.skip("no hipcc")
    source = tmp_path / "rows.hip"
    source.write_text(PROGRAM)
    done = subprocess.run([HIPCC, "--offload-arch=gfx950", "--cuda-host-only", "-fsyntax-only", "-std=c++17", "-I", os.path.join(REPO, "include"),
                           "-I", os.path.join(REPO, "lmserve_amd", "csrc"), str(source)], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-3000:]
