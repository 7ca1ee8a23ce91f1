"""The kernels over a vocabulary, compiled for the host with AddressSanitizer and run lane by lane: what they read and
write lies inside the arrays they are given, lanes stay together where the wave acts as one, and the best columns are
those of a sort."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "theano_amd", "csrc")
CLANG = shutil.which("clang++", path="/opt/rocm/llvm/bin:/opt/rocm/lib/llvm/bin") or shutil.which("clang++")


def between(text, first, last):
    at = text.index(first)
    return text[at:text.index(last, at)]


def device_code():
    """The device half of the sources as one text of plain C++."""
    def read(*name):
        with open(os.path.join(CSRC, *name)) as f:
            return f.read()

    common, rows, vocab = read("kernels", "thx_common.h"), read("thx_rows_device.h"), read("thx_vocab.cpp")
    parts = [between(common, "typedef unsigned char thx_bool", "#ifndef INFINITY"), "#define THX_DEV inline\nnamespace thx {\n",
             between(common, "template <int B> struct AlignFor", "// Sums over the V float16 elements"), "}\n",
             rows[rows.index("namespace thx {"):],
             between(vocab, "namespace thx {", "int acc_code(int dtype)"), "}\n}\n"]
    # barriers to the compiler's view of registers, which name the device's
    return re.sub(r"asm volatile\([^;]*\);", ";", "".join(parts))


@pytest.mark.skipif(CLANG is None, reason="no compiler with half precision for the host")
def test_best_columns_lane_by_lane(tmp_path):
    kernels, program = tmp_path / "vocab_kernels.h", str(tmp_path / "vocab_host")
    kernels.write_text(device_code())
    cmd = [CLANG, "-std=c++17", "-O1", "-g1", "-march=native", "-w", "-Xarch_host", "-fsanitize=address",
           "-DVOCAB_KERNELS=\"%s\"" % kernels, os.path.join(ROOT, "tests", "native", "vocab_host.cpp"), "-o", program]
    res = subprocess.run(cmd, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    env = dict(os.environ, ASAN_OPTIONS="detect_stack_use_after_return=0:detect_leaks=0")
    env.pop("LD_PRELOAD", None)
    res = subprocess.run([program], capture_output=True, text=True, env=env, timeout=600)
    assert res.returncode == 0, res.stdout[-4000:] + res.stderr[-4000:]
    assert " 0 wrong" in res.stdout
