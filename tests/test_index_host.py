"""The kernels' index arithmetic at the ends of 32 bits, compiled for the host (csrc/index.cuh): signed overflow ends
the program."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rubidium-train_b200", "csrc")

pytestmark = pytest.mark.skipif(shutil.which("g++") is None, reason="no g++")


def run(tmp_path, body):
    src = tmp_path / "t.cpp"
    src.write_text('#include <cstdio>\n#include "index.cuh"\nusing namespace rbk;\nint main() {\n' + body + "\n}\n")
    exe = tmp_path / "t"
    subprocess.run(["g++", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I", CSRC, str(src), "-o",
                    str(exe)], check=True)
    return [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]


def test_token_at_the_end(tmp_path):
    """The token that a lane looks up, behind a warp's last one too, is one of the call's: also with 2^31 - 1 of them."""
    cases = [(tk, sub, n) for n in (1, 2, 7, 2 ** 31 - 2, 2 ** 31 - 1) for sub in (0, 1)
             for tk in {0, 1, n - 2, n - 1, n} if 0 <= tk <= n]
    body = "volatile int v;\n" + "".join(
        f'v = {tk}; printf("%d\\n", token_at(v, {sub}, {n}));\n' for tk, sub, n in cases) + "return 0;"
    assert run(tmp_path, body) == [min(tk + sub, n - 1) for tk, sub, n in cases]


def test_tokens_are_looked_up_through_it():
    src = open(os.path.join(CSRC, "qk.cu")).read()
    assert src.count("token_at(tk, sub, p.tokens)") == 2 and "min(tk + sub" not in src
